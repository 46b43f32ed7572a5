"""ctypes binding of libpsquant.so (the gfx950 HIP kernels behind the C ABI in include/psquant.h).

The library is built in-tree by ``build_lib.py`` into ``lib/libpsquant.so``.  There is no
fallback implementation: if the library is missing, ``lib()`` raises :class:`NativeLibraryError`
(an ``ImportError``, deliberately *not* one of the exception types QuantLinear's native branch
turns into a warn-and-dequantize fallback), so a broken install fails loudly.

The reference loads its own native helper the same way -- a runtime-built ``.so`` with
``extern "C"`` entry points (powershard/ats_memory.py:80-91, ats_allocator.cpp:14-52).
"""
import ctypes
import importlib.util
import os
import sys
import threading
import warnings
from pathlib import Path

DIRECT_PATH = Path(__file__).resolve().parent / "lib" / "psq_direct.so"
LIB_PATH = Path(os.environ.get("PSQUANT_LIB", Path(__file__).resolve().parent / "lib" / "libpsquant.so"))
ABI_VERSION = 1

BF16, F16, F32 = 0, 1, 2
W_UINT4, W_INT8 = 0, 1   # enum psq_weight_kind
Q8_I8, Q8_E4M3, Q8_E5M2 = 0, 1, 2   # enum psq_q8_weights
CODES_NONE, CODES_I8, CODES_E4M3 = 0, 1, 2   # enum psq_codes

# Every exported entry point: name -> (restype, argtypes).  Mirrors include/psquant.h.
_P, _I64, _I, _F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
SIGNATURES = {
    "psq_abi_version": (_I, []),
    "psq_last_error": (ctypes.c_char_p, []),
    "psq_device_supported": (_I, [_I]),
    "psq_quantize_rows_i8": (_I, [_P, _I, _I64, _I64, _I64, _I, _P, _P, _I64, _P, _P]),
    "psq_quantize_rows_fp8": (_I, [_P, _I, _I64, _I64, _I64, _I, _P, _P, _I64, _P, _P]),
    "psq_rotate_rows": (_I, [_P, _I, _I64, _I64, _I64, _I, _P, _I, _I64, _P]),
    "psq_gemm_i8": (_I, [_P, _I64, _P, _P, _I64, _P, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_gemm_i8_act": (_I, [_P, _I64, _P, _P, _I64, _P, _P, _I, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_gemm_i8_i32": (_I, [_P, _I64, _P, _I64, _P, _I64, _I64, _I64, _I64, _P]),
    "psq_gemm_i8_8wave": (_I, [_P, _I64, _P, _P, _I64, _P, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_gemm_fp8": (_I, [_P, _I64, _P, _P, _I64, _P, _I, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_gemm_fp8_e5m2w": (_I, [_P, _I64, _P, _P, _I64, _P, _I, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_gemm_fp8_act": (_I, [_P, _I64, _P, _P, _I64, _P, _I, _P, _I, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_linear_q8_scratch_bytes": (_I64, [_I64, _I64]),
    "psq_linear_q8": (_I, [_I, _P, _I, _I64, _I, _P, _I64, _P, _I, _P, _I, _I, _P, _I, _I64, _I64, _I64, _I64, _P, _P]),
    "psq_gemm_w4a16": (_I, [_P, _I, _I64, _P, _P, _P, _I, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_gemm_w8a16": (_I, [_P, _I, _I64, _P, _P, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_gemm_wonly_workspace_bytes": (_I64, [_I, _I64, _I64, _I64, _I64, _I]),
    "psq_gemm_w4a16_ws": (_I, [_P, _I, _I64, _P, _P, _P, _I, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P, _I64, _P]),
    "psq_gemm_w8a16_ws": (_I, [_P, _I, _I64, _P, _P, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P, _I64, _P]),
    "psq_linear_w8a16": (_I, [_P, _I, _I64, _I, _P, _P, _P, _I, _P, _I64, _I64, _I64, _I64, _P, _P, _I64, _P,
                              ctypes.c_uint64, _P]),
    "psq_gemm_w4a16_noalloc": (_I, [_P, _I, _I64, _P, _P, _P, _I, _P, _I, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "psq_dequant_uint4": (_I, [_P, _P, _P, _I, _I64, _I64, _P, _I, _P]),
    "psq_dequant_i8_rows": (_I, [_P, _P, _I64, _I64, _I, _P, _I, _P]),
    "psq_dequant_fp8": (_I, [_P, _P, _I, _I64, _I64, _P, _I, _P]),
    "psq_dequant_e5m2": (_I, [_P, _P, _I, _I64, _I64, _P, _I, _P]),
    "psq_add_rms_norm": (_I, [_I, _P, _I, _I64, _P, _I64, _P, _I, _F, _P, _I64, _I, _P, _P, _I64, _P, _I64, _I64, _P]),
    "psq_kv_write": (_I, [_I, _P, _P, _I, _I64, _I64, _I64, _I64, _P, _I64, _I, _I, _P, _P, _P, _P, _I64, _I, _P]),
    "psq_kv_read": (_I, [_I, _P, _I64, _P, _P, _I, _P, _P, _I64, _I, _I, _I, _P, _P, _I, _P]),
    "psq_paged_attention_workspace_bytes": (_I64, [_I, _I64, _I, _I, _I, _I64]),
    "psq_paged_attention_own_workspace": (_I, [_I, _I64, _I, _I, _I, _I64]),
    "psq_paged_attention": (_I, [_I, _P, _I, _I64, _I64, _P, _P, _P, _P, _I64, _I, _P, _I64, _I64, _P, _I64, _I, _I, _I, _F,
                                 _I64, _I64, _P, _P, _P, _I64, _P]),
    "psq_flag_nonfinite": (_I, [_P, _I, _I64, _P, ctypes.c_uint64, _P]),
}

DIRECT_CALLS = ("psq_add_rms_norm", "psq_kv_write", "psq_kv_read", "psq_paged_attention_workspace_bytes",
                "psq_paged_attention_own_workspace", "psq_paged_attention")


class NativeLibraryError(ImportError):
    """libpsquant.so is missing or unusable: the native path cannot run."""


_lock = threading.Lock()
_lib = None


def lib():
    """The loaded library (loaded once, thread-safe).  Raises NativeLibraryError if absent."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise NativeLibraryError(
                    f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                    "or comfyui-powershard_amd/powershard_amd/build_lib.py")
            try:
                handle = ctypes.CDLL(str(LIB_PATH))
            except OSError as error:
                raise NativeLibraryError(f"cannot load {LIB_PATH}: {error}") from error
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(handle, name)
                fn.restype, fn.argtypes = res, args
            if handle.psq_abi_version() != ABI_VERSION:
                raise NativeLibraryError(f"{LIB_PATH}: ABI {handle.psq_abi_version()} != {ABI_VERSION}")
            _lib = handle
    return _lib


_direct = None


def direct():
    """The module of the decoder operators' direct calls (csrc/direct.cpp), bound to the loaded library, or
    False where it cannot be used: it belongs to one release of torch and of Python, and the calls that it
    shortens work without it.  A missing or foreign module is named in one warning."""
    global _direct
    if _direct is None:
        handle = lib()
        with _lock:
            if _direct is None:
                _direct = _load_direct(handle)
    return _direct


def _load_direct(handle):
    import torch
    try:
        spec = importlib.util.spec_from_file_location("psq_direct", DIRECT_PATH)
        module = importlib.util.module_from_spec(spec)
        if module.TORCH_VERSION != torch.__version__.split("+")[0]:
            raise ImportError(f"built for torch {module.TORCH_VERSION}, this is {torch.__version__}")
        if module.PYTHON_VERSION != sys.hexversion >> 16:
            raise ImportError(f"built for Python {module.PYTHON_VERSION >> 8}.{module.PYTHON_VERSION & 255}, this is {sys.version.split()[0]}")
        module.bind({name: ctypes.cast(getattr(handle, name), ctypes.c_void_p).value for name in DIRECT_CALLS})
    except ImportError as error:
        warnings.warn(f"psquant: {DIRECT_PATH} is not used ({error}): the decoder operators' calls take longer", stacklevel=4)
        return False
    return module


def available():
    try:
        lib()
        return True
    except NativeLibraryError:
        return False


def last_error():
    return lib().psq_last_error().decode("utf-8", "replace")


def check(status, what):
    """Turn a non-zero status into RuntimeError (the type QuantLinear's fallback handles)."""
    if status != 0:
        raise RuntimeError(f"psquant {what} failed ({status}): {last_error()}")
