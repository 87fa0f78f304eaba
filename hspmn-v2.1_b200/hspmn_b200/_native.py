"""ctypes binding of libhspmn_sm100.so (C ABI in include/hspmn_sm100.h).

The library is loaded from this package directory only; there is no other
implementation to fall back to, so every entry point raises when the library
is missing or the device is not a B200.
"""

from __future__ import annotations

import ctypes
import os
import threading

LIB_NAME = "libhspmn_sm100.so"
LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), LIB_NAME)
TORCH_LIB_PATH = os.path.join(os.path.dirname(LIB_PATH), "libhspmn_torch.so")

HSPMN_F32, HSPMN_F16, HSPMN_BF16 = 0, 1, 2
DEVERR_POSITION, DEVERR_UNSORTED, DEVERR_TIMEOUT, DEVERR_PAGE = 1, 2, 4, 8

# name -> (restype, argtypes)
_i64 = ctypes.c_int64
_vp = ctypes.c_void_p
_int = ctypes.c_int
_SIGNATURES = {
    "hspmn_version": (_int, []),
    "hspmn_strerror": (ctypes.c_char_p, [_int]),
    "hspmn_router_topk": (_int, [_vp, _int, _i64, _vp, _int, _int, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp]),
    "hspmn_gate_logits": (_int, [_vp, _int, _i64, _i64, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _vp]),
    "hspmn_gather_rows": (_int, [_vp, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _vp]),
    "hspmn_scatter_rows": (_int, [_vp, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _vp]),
    "hspmn_sqdk_fwd": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _vp,
                              _i64, _i64, _i64, _i64, _i64, _i64, _int, ctypes.c_float,
                              _vp, ctypes.c_size_t, _vp]),
    "hspmn_sqdk_workspace_size": (_i64, [_i64, _i64, _i64, _i64, _i64, _i64]),
    "hspmn_sqdk_fwd_noalloc": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _vp,
                                      _i64, _i64, _i64, _i64, _i64, _i64, _int, ctypes.c_float, _vp]),
    "hspmn_sqdk_fwd_lse": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _i64, _i64,
                                  _i64, _i64, _i64, _i64, _i64, _i64, _int, ctypes.c_float,
                                  _vp, ctypes.c_size_t, _vp]),
    "hspmn_sqdk_bwd_workspace_size": (_i64, [_i64, _i64, _i64, _i64]),
    "hspmn_sqdk_bwd": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _i64,
                              _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _int,
                              ctypes.c_float, _vp, ctypes.c_size_t, _vp]),
    "hspmn_rope_gather_rows": (_int, [_vp, _i64, _i64, _int, _vp, _i64, _vp, _vp, _i64, _vp, _i64, _i64,
                                      _i64, _i64, _i64, _i64, _i64, _int, _vp]),
    "hspmn_rope_rows": (_int, [_vp, _i64, _i64, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _i64,
                               _i64, _int, _vp]),
    "hspmn_scatter_add_rows": (_int, [_vp, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
                                      _int, _vp]),
    "hspmn_paged_slots": (_int, [_vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _vp,
                                 _vp]),
    "hspmn_rope_paged_write": (_int, [_vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _i64, _i64, _int, _vp, _vp,
                                      _vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64,
                                      _int, _vp]),
    "hspmn_sqdk_paged_workspace_size": (_i64, [_i64, _i64, _i64, _i64, _i64]),
    "hspmn_sqdk_paged_fwd": (_int, [_vp, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _vp,
                                    _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _int,
                                    ctypes.c_float, _i64, _vp, ctypes.c_size_t, _vp]),
    "hspmn_device_errors": (_int, [ctypes.POINTER(ctypes.c_uint), _int, _vp]),
}
EXPORTED = tuple(_SIGNATURES)

_lib = None
_lock = threading.Lock()


class HSPMNNativeError(RuntimeError):
    """A library entry point returned a non-zero status."""


def available() -> bool:
    return os.path.exists(LIB_PATH)


def lib() -> ctypes.CDLL:
    """Load (once) and return the native library; raise if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"{LIB_NAME} is not built (expected at {LIB_PATH}); run "
                    "`python hspmn-v2.1_b200/build_native.py` on a machine with the CUDA toolkit")
            handle = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in _SIGNATURES.items():
                fn = getattr(handle, name)
                fn.restype = res
                fn.argtypes = args
            _lib = handle
    return _lib


def torch_build_id() -> str:
    """What libhspmn_torch.so must have been built for, as it stands in the file."""
    import sysconfig
    import torch
    return (f"hspmn_torch for torch {torch.__version__}, C++ ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, "
            f"{sysconfig.get_config_var('SOABI')};")


def built_for_this_torch(path: str) -> bool:
    with open(path, "rb") as f:
        return torch_build_id().encode() in f.read()


def load_torch_ops():
    """Load libhspmn_torch.so: its operators are then registered with PyTorch.
    Returns it as a Python module; raises if it is not built, or not for this
    PyTorch."""
    if not os.path.exists(TORCH_LIB_PATH):
        raise RuntimeError(
            f"{os.path.basename(TORCH_LIB_PATH)} is not built (expected at {TORCH_LIB_PATH}); run "
            "`python hspmn-v2.1_b200/build_native.py` on a machine with the CUDA toolkit")
    import importlib.machinery
    import importlib.util
    import torch  # noqa: F401 (the module links against its libraries)
    lib()
    if not built_for_this_torch(TORCH_LIB_PATH):
        raise RuntimeError(
            f"{TORCH_LIB_PATH} was not built for PyTorch {torch.__version__} and this Python; run "
            "`python hspmn-v2.1_b200/build_native.py` on a machine with the CUDA toolkit")
    loader = importlib.machinery.ExtensionFileLoader("libhspmn_torch", TORCH_LIB_PATH)
    try:
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("libhspmn_torch", loader))
        loader.exec_module(module)
    except ImportError as e:
        raise RuntimeError(
            f"{TORCH_LIB_PATH} does not load with PyTorch {torch.__version__} ({e}); run "
            "`python hspmn-v2.1_b200/build_native.py --force` on a machine with the CUDA toolkit") from e
    return module


def strerror(status: int) -> str:
    return lib().hspmn_strerror(int(status)).decode()


def check(status: int, what: str) -> None:
    if status != 0:
        raise HSPMNNativeError(f"{what} failed: {strerror(status)} (status {status})")


def device_errors(stream: int = 0, clear: bool = True) -> int:
    """Synchronise ``stream`` and return the device flag word (DEVERR_* bits)."""
    bits = ctypes.c_uint(0)
    check(lib().hspmn_device_errors(ctypes.byref(bits), int(clear), ctypes.c_void_p(stream)),
          "hspmn_device_errors")
    return int(bits.value)


def i64_array(vals):
    arr = (ctypes.c_int64 * len(vals))(*[int(v) for v in vals])
    return arr
