"""ctypes binding of libmce.so (declarations in include/mce.h), libmce_attn.so (include/mce_attn.h, mce_paged.h,
mce_rope.h) and libmce_serve.so (include/mce_pack.h, mce_cache.h).

torch is imported before the library is loaded: torch ships its own libamdhip64.so with the same SONAME as
/opt/rocm's, so loading torch first makes libmce.so bind to the one HIP runtime that owns torch's streams
and allocations.
"""
import ctypes
import os

import torch  # noqa: F401  (must precede the CDLL load, see module docstring)

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libmce.so")
ATTN_LIB_PATH = os.path.join(HERE, "libmce_attn.so")
SERVE_LIB_PATH = os.path.join(HERE, "libmce_serve.so")

_P = ctypes.c_void_p
_F = ctypes.c_float
_I = ctypes.c_int64
_S = ctypes.c_size_t
_INT = ctypes.c_int

# name -> (restype, argtypes); kept in the order of include/mce.h, include/mce_induct.h, include/mce_swiglu.h
SIGNATURES = {
    "mce_version": (_INT, []),
    "mce_error_string": (ctypes.c_char_p, [_INT]),
    "mce_last_hip_error": (_INT, []),
    "mce_fwd_ws_bytes": (_S, [_I, _I, _I]),
    "mce_fwd": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _S, _P]),
    "mce_fwd_noalloc": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P]),
    "mce_fwd_sparse": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _INT, _I, _I, _I, _I, _P, _P, _P, _P, _P, _S, _P]),
    "mce_bwd_ws_bytes": (_S, [_I, _I, _I]),
    "mce_bwd_logits_grad": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P, _P, _P, _S, _P]),
    "mce_bwd_logits_grad_sparse": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _INT, _P, _P, _P, _I, _I, _I, _I, _P, _P,
                                          _P, _S, _P]),
    "mce_lse_fwd": (_INT, [_P, _I, _P, _I, _P, _P, _I, _I, _I, _I, _P, _P, _P, _S, _P]),
    "mce_bwd_lse_grad": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P, _P, _S, _P]),
    "mce_bwd_dhidden": (_INT, [_P, _I, _I, _I, _I, _P, _INT, _I, _P, _S, _P]),
    "mce_bwd_dweight": (_INT, [_P, _I, _I, _I, _I, _P, _I, _P, _S, _P]),
    "mce_bwd": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P, _INT, _I, _P, _I, _P, _P, _P,
                       _S, _P]),
    "mce_bwd_block_rows": (_I, [_I, _I, _I, _I]),
    "mce_bwd_blocked_ws_bytes": (_S, [_I, _I, _I, _I]),
    "mce_bwd_blocked": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _INT, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _INT, _I,
                               _P, _I, _P, _P, _P, _P, _S, _P]),
    "mce_bwd_lse_blocked": (_INT, [_P, _I, _P, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _INT, _I, _P, _I, _P,
                                   _P, _S, _P]),
    "mce_train_ws_bytes": (_S, [_I, _I, _I, _I]),
    "mce_train_block_rows": (_I, [_I, _I, _I, _I]),
    "mce_fwd_train": (_INT, [_P, _I, _P, _I, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _INT, _P, _P, _P, _P, _P,
                             _P, _INT, _I, _P, _I, _P, _P, _S, _P]),
    "mce_fwd_train_sparse": (_INT, [_P, _I, _P, _I, _P, _I, _P, _P, _P, _P, _INT, _I, _I, _I, _I, _I, _INT, _P, _P,
                                    _P, _P, _P, _INT, _I, _P, _I, _P, _P, _S, _P]),
    "mce_bwd_train": (_INT, [_P, _I, _P, _P, _I, _I, _I, _I, _P, _P, _P, _P, _INT, _I, _P, _I, _P, _P, _P, _S, _P]),
    "mce_bwd_train_dcval": (_INT, [_P, _P, _P, _INT, _P, _P, _P, _I, _I, _I, _I, _I, _P, _P, _S, _P]),
    "mce_train_flagged": (_INT, [_P, _I, _I, _I, _I, _P, _P]),
    "mce_train_target_logits": (_INT, [_P, _I, _I, _I, _I, _P, _P]),
    "mce_bwd_lse_train": (_INT, [_P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _INT, _I, _P, _I, _P, _P, _S, _P]),
    "mce_train_set_threshold": (None, [ctypes.c_float]),
    "mce_prof_start": (_INT, []),
    "mce_prof_stop": (_INT, [_P, _P, _INT]),
    # include/mce_induct.h
    "mce_induct": (_INT, [_P, _I, _I, _INT, _INT, _P, _I, _I, _P, _P, _P, _P, _P, _P]),
    "mce_induct_max_len": (_INT, []),
    "mce_induct_ws_bytes": (_S, [_I, _I, _INT]),
    "mce_induct_ws": (_INT, [_P, _I, _I, _INT, _INT, _P, _I, _I, _P, _P, _P, _P, _P, _P, _S, _P]),
    # include/mce_swiglu.h
    "mce_swiglu_fwd": (_INT, [_P, _I, _I, _INT, _P, _P]),
    "mce_swiglu_bwd": (_INT, [_P, _P, _INT, _I, _I, _INT, _P, _P]),
    "mce_swiglu_last_hip_error": (_INT, []),
}

# the attention library, in the order of include/mce_attn.h, include/mce_paged.h, include/mce_rope.h
_TENSOR = [_P, _I, _I, _I]   # pointer and element strides (batch, token, head)
ATTN_SIGNATURES = {
    "mce_attn_error_string": (ctypes.c_char_p, [_INT]),
    "mce_attn_last_hip_error": (_INT, []),
    "mce_attn_fwd": (_INT, 3 * _TENSOR + [_P] + 7 * [_I] + [_F, _INT, _P, _P, _P, _P]),
    "mce_attn_bwd_ws_bytes": (_S, 7 * [_I]),
    "mce_attn_bwd": (_INT, 4 * _TENSOR + [_P] + 7 * [_I] + [_F, _INT, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    # include/mce_paged.h
    "mce_paged_ws_bytes": (_S, 8 * [_I]),
    "mce_paged": (_INT, [_P, _I, _I] + 2 * _TENSOR + [_P, _I, _P] + 9 * [_I] + [_F, _INT, _P, _P, _S, _P]),
    # include/mce_rope.h
    "mce_rope_fwd": (_INT, 2 * _TENSOR + [_P, _P, _I, _P, _INT, _I, _I, _P, _P] + 6 * [_I] +
                     [_INT, _F, _INT, _INT, _P, _P, _P]),
    "mce_rope_bwd_ws_bytes": (_S, 5 * [_I] + [_INT]),
    "mce_rope_bwd": (_INT, 4 * _TENSOR + [_P, _P, _I, _P, _INT, _I, _I, _P, _P] + 6 * [_I] +
                     [_INT, _F, _INT, _INT, _P, _P, _P, _P, _P, _S, _P]),
}

# the library of packed sequences and of the 8-bit cache, in the order of include/mce_pack.h, include/mce_cache.h
_ROWS = [_P, _I, _I]   # pointer and element strides (token, head)
SERVE_SIGNATURES = {
    "mce_serve_error_string": (ctypes.c_char_p, [_INT]),
    "mce_serve_last_hip_error": (_INT, []),
    "mce_pack_plan_bytes": (_S, 8 * [_I]),
    "mce_pack_fwd_ws_bytes": (_S, 8 * [_I]),
    "mce_pack_fwd": (_INT, 3 * _ROWS + [_P, _P] + 8 * [_I] + [_F, _INT, _P, _P, _P, _P, _S, _P, _S, _P]),
    "mce_pack_bwd_ws_bytes": (_S, 8 * [_I]),
    "mce_pack_bwd": (_INT, 4 * _ROWS + [_P, _P] + 8 * [_I] + [_F, _INT, _P, _P, _P, _P, _P, _P, _P, _P, _S, _P]),
    # include/mce_cache.h
    "mce_cache_write": (_INT, 2 * _ROWS + 2 * _TENSOR + [_P, _P, _P, _I, _P, _P] + 8 * [_I] + [_INT, _P]),
    "mce_cache_read": (_INT, 2 * _TENSOR + [_P, _P, _P, _I, _P] + 8 * [_I] + [_INT, _P, _P, _P]),
    "mce_cache_attn_ws_bytes": (_S, 8 * [_I]),
    "mce_cache_attn": (_INT, [_P, _I, _I] + 2 * _TENSOR + [_P, _P, _P, _I, _P] + 10 * [_I] + [_F, _INT, _P, _P, _S, _P]),
}

_lib = None
_attn_lib = None
_serve_lib = None
_call_hook = None  # optional callable(name, phase) run around every C-ABI call, phase "begin" / "end"


class MceError(RuntimeError):
    pass


def _load(path, signatures):
    if not os.path.exists(path):
        raise MceError(f"{path} is missing; build it with `python -m memarch_amd.build`")
    lib = ctypes.CDLL(path)
    for name, (res, args) in signatures.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


def load():
    """Load libmce.so once. Raises if the library has not been built: there is no fallback path."""
    global _lib
    if _lib is None:
        _lib = _load(LIB_PATH, SIGNATURES)
    return _lib


def load_attn():
    """Load libmce_attn.so once. Raises if the library has not been built: there is no fallback path."""
    global _attn_lib
    if _attn_lib is None:
        _attn_lib = _load(ATTN_LIB_PATH, ATTN_SIGNATURES)
    return _attn_lib


def load_serve():
    """Load libmce_serve.so once. Raises if the library has not been built: there is no fallback path."""
    global _serve_lib
    if _serve_lib is None:
        _serve_lib = _load(SERVE_LIB_PATH, SERVE_SIGNATURES)
    return _serve_lib


def check(rc, what):
    if rc != 0:
        if what in SERVE_SIGNATURES:
            lib = load_serve()
            msg = lib.mce_serve_error_string(rc).decode()
            raise MceError(f"{what} failed: {msg} (code {rc}, hipError {lib.mce_serve_last_hip_error()})")
        if what in ATTN_SIGNATURES:
            lib = load_attn()
            msg = lib.mce_attn_error_string(rc).decode()
            raise MceError(f"{what} failed: {msg} (code {rc}, hipError {lib.mce_attn_last_hip_error()})")
        lib = load()
        msg = lib.mce_error_string(rc).decode()
        hip = lib.mce_last_hip_error()
        raise MceError(f"{what} failed: {msg} (code {rc}, hipError {hip})")


def set_call_hook(fn):
    """Install fn(name, phase) to be called just before ("begin") and after ("end") every C-ABI call (e.g. to
    record stream events around each stage); returns the previous hook. None removes it."""
    global _call_hook
    prev, _call_hook = _call_hook, fn
    return prev


def call(name, *args):
    hook = _call_hook
    if hook is not None:
        hook(name, "begin")
    lib = load_serve() if name in SERVE_SIGNATURES else load_attn() if name in ATTN_SIGNATURES else load()
    check(getattr(lib, name)(*args), name)
    if hook is not None:
        hook(name, "end")
