"""ctypes binding of the C ABI in include/dion_lm.h (libdion_lm.so).

The library is built in-tree by `python __graft_entry__.py` (hipcc, gfx950), like the codec's
(`_lib.py`), whose error classes it shares.  There is no CPU or PyTorch fallback for its operators.
"""
from __future__ import annotations

import ctypes
import hashlib
import os

from ._lib import DionLibraryError, DionUnsupportedError, DION_E_UNSUPPORTED, DION_OK

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "csrc", "libdion_lm.so")
SOURCE_DIR = os.path.join(HERE, "csrc", "lm")
HEADERS = tuple(os.path.join(os.path.dirname(HERE), "include", n) for n in ("dion_codec.h", "dion_lm.h"))
ABI_VERSION = 1

DTYPE_E4M3 = 3
XENT_FORWARD = 1
XENT_BACKWARD = 2

# every symbol include/dion_lm.h declares
EXPORTED = (
    "dion_lm_abi_version",
    "dion_lm_build_id",
    "dion_lm_last_error",
    "dion_dropout_add",
    "dion_rms_norm_add",
    "dion_rms_norm_add_workspace_bytes",
    "dion_rms_norm_add_backward",
    "dion_xent_workspace_bytes",
    "dion_xent_forward",
    "dion_xent_backward",
)


def source_build_id() -> str | None:
    """SHA-256 (16 hex digits) over csrc/lm/*.hip, csrc/lm/*.hpp and the two headers, by file name
    then bytes, sorted by name; None when the sources are absent."""
    if not os.path.isdir(SOURCE_DIR) or not all(os.path.exists(h) for h in HEADERS):
        return None
    files = [(n, os.path.join(SOURCE_DIR, n)) for n in os.listdir(SOURCE_DIR) if n.endswith((".hip", ".hpp"))]
    files += [(os.path.basename(h), h) for h in HEADERS]
    h = hashlib.sha256()
    for name, path in sorted(files):
        h.update(name.encode() + b"\0")
        with open(path, "rb") as fh:
            h.update(fh.read() + b"\0")
    return h.hexdigest()[:16]


class DionRng(ctypes.Structure):
    _fields_ = [("seed", ctypes.c_uint64), ("offset", ctypes.c_uint64), ("device", ctypes.c_void_p)]


class DionNormDesc(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("cols", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("w_dtype", ctypes.c_int32), ("gw_dtype", ctypes.c_int32), ("y_dtype", ctypes.c_int32),
                ("scale_block", ctypes.c_int32), ("accumulate", ctypes.c_int32), ("eps", ctypes.c_float),
                ("p", ctypes.c_double)] + [
        (n, ctypes.c_int64) for n in ("ld_x", "ld_residual", "ld_h", "ld_y", "ld_grad_y", "ld_grad_h", "ld_grad_x",
                                      "ld_grad_residual")]


class DionXentDesc(ctypes.Structure):
    _fields_ = [("tokens", ctypes.c_int64), ("hidden", ctypes.c_int32), ("vocab", ctypes.c_int32),
                ("dtype", ctypes.c_int32), ("gw_dtype", ctypes.c_int32), ("accumulate", ctypes.c_int32),
                ("pack_weight", ctypes.c_int32), ("vocab_start", ctypes.c_int64), ("vocab_total", ctypes.c_int64),
                ("ignore_index", ctypes.c_int64), ("ld_hidden", ctypes.c_int64), ("ld_weight", ctypes.c_int64),
                ("ld_grad_hidden", ctypes.c_int64), ("ld_grad_weight", ctypes.c_int64), ("piece_bytes", ctypes.c_int64)]


_P = ctypes.c_void_p
_NORM = ctypes.POINTER(DionNormDesc)
_XENT = ctypes.POINTER(DionXentDesc)
_RNG = ctypes.POINTER(DionRng)
_SIZE = ctypes.POINTER(ctypes.c_size_t)
_I64 = ctypes.c_int64

_SIGNATURES = {
    "dion_lm_abi_version": ([], ctypes.c_int),
    "dion_lm_build_id": ([], ctypes.c_char_p),
    "dion_lm_last_error": ([], ctypes.c_char_p),
    "dion_dropout_add": ([_I64, _I64, ctypes.c_int32, _P, _I64, _P, _I64, _P, _I64, ctypes.c_double, _RNG, _P],
                         ctypes.c_int),
    "dion_rms_norm_add": ([_NORM, _P, _P, _P, _P, _P, _P, _P, _RNG, _P], ctypes.c_int),
    "dion_rms_norm_add_workspace_bytes": ([_NORM, _SIZE], ctypes.c_int),
    "dion_rms_norm_add_backward": ([_NORM, _P, _P, _P, _P, _P, _P, _P, _P, _RNG, _P, ctypes.c_size_t, _P],
                                   ctypes.c_int),
    "dion_xent_workspace_bytes": ([_XENT, ctypes.c_int, _SIZE], ctypes.c_int),
    "dion_xent_forward": ([_XENT, _P, _P, _P, _P, _P, _P, _P, ctypes.c_size_t, _P], ctypes.c_int),
    "dion_xent_backward": ([_XENT, _P, _P, _P, _P, _P, _P, _P, _P, ctypes.c_size_t, _P], ctypes.c_int),
}

_lib = None


def load(path: str = LIB_PATH):
    """Load (once) and return the library; raise if it is missing or stale."""
    global _lib
    if _lib is not None and path == LIB_PATH:
        return _lib
    if not os.path.exists(path):
        raise DionLibraryError(
            f"[DION_HIP_LIBRARY_MISSING] {path} not found; build it with "
            "`python __graft_entry__.py` (hipcc --offload-arch=gfx950). There is no CPU fallback.")
    lib = ctypes.CDLL(path)
    for name, (args, res) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    ver = lib.dion_lm_abi_version()
    if ver != ABI_VERSION:
        raise DionLibraryError(f"[DION_HIP_ABI_MISMATCH] library ABI {ver}, expected {ABI_VERSION}")
    want, got = source_build_id(), lib.dion_lm_build_id().decode("ascii", "replace")
    if path == LIB_PATH and want is not None and got != want:
        raise DionLibraryError(
            f"[DION_HIP_LIBRARY_STALE] {path} was built from sources {got}, the tree holds {want}; rebuild it "
            "with `python __graft_entry__.py`")
    if path == LIB_PATH:
        _lib = lib
    return lib


def check(rc: int, what: str) -> None:
    if rc != DION_OK:
        msg = load().dion_lm_last_error().decode("utf-8", "replace")
        cls = DionUnsupportedError if rc == DION_E_UNSUPPORTED else DionLibraryError
        err = cls(f"[DION_HIP_ERROR] {what} failed ({rc}): {msg}")
        err.code = rc
        raise err
