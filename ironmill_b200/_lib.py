"""ctypes binding of libironmill_cuda.so (the C ABI declared in include/ironmill_cuda.h).

There is no fallback: if the library is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libironmill_cuda.so")

IM_OK = 0
IM_DTYPE_F16 = 0
IM_DTYPE_F32 = 1
IM_DTYPE_BF16 = 2

STATUS_NAMES = {
    0: "IM_OK", -1: "IM_ERR_INVALID", -2: "IM_ERR_CUDA", -3: "IM_ERR_ALLOC", -4: "IM_ERR_BOUNDS",
    -5: "IM_ERR_TIMEOUT", -6: "IM_ERR_NCCL", -7: "IM_ERR_STATE", -8: "IM_ERR_NO_DEVICE",
}


class CudaSysError(RuntimeError):
    """Counterpart of MetalSysError (crates/ironmill-metal-sys/src/error.rs:5-41)."""

    def __init__(self, code: int, message: str):
        super().__init__(f"{STATUS_NAMES.get(code, code)}: {message}")
        self.code = code
        self.message = message


_lib = None

_VOIDP_RESTYPE = ("im_cuda_buffer_ptr",)
_SIZE_RESTYPE = ("im_cuda_device_allocated_bytes", "im_cuda_buffer_length", "im_cuda_affine_weight_bytes",
                 "im_cuda_model_memory_bytes", "im_cuda_model_step_bytes", "im_cuda_tq_scratch_bytes",
                 "im_cuda_sdpa_f16_scratch_bytes", "im_cuda_tq_prefill_scratch_bytes",
                 "im_cuda_paged_attention_scratch_bytes", "im_cuda_paged_prefix_attention_scratch_bytes",
                 "im_cuda_paged_attention_weights_scratch_bytes", "im_cuda_beam_select_scratch_bytes")
_VOID_RESTYPE = ("im_cuda_device_free", "im_cuda_buffer_free", "im_cuda_affine_weight_free", "im_cuda_model_free",
                 "im_cuda_tq_free", "im_cuda_tp_free")

_P, _I, _L, _F, _Z = C.c_void_p, C.c_int, C.c_int64, C.c_float, C.c_size_t
# Calls between two forwards are short: with their argument types known, plain numbers and addresses are passed.
_ARGTYPES = {
    "im_cuda_paged_append": (_P, _P, _I, _P, _L, _P, _L, _P, _I, _P, _L, _P, _L, _I, _P, _P, _I, _I, _I, _I, _P, _P),
    "im_cuda_paged_append_normed": (_P, _P, _P, _P),
    "im_cuda_paged_attention_scratch_bytes": (_P, _P, _I, _I, _I),
    "im_cuda_paged_attention": (_P, _P, _I, _P, _L, _P, _L, _I, _P, _I, _I, _P, _I, _F, _I, _P, _Z, _P),
    "im_cuda_paged_prefix_attention_scratch_bytes": (_P, _P, _I, _I, _I, _I),
    "im_cuda_paged_prefix_attention": (_P, _P, _P, _P),
    "im_cuda_paged_attention_weights_scratch_bytes": (_P, _P, _I, _I, _I),
    "im_cuda_paged_attention_weights": (_P, _P, _P, _P),
    "im_cuda_paged_evict": (_P, _P, _P, _P),
    "im_cuda_paged_keep": (_P, _P, _P, _I, _P, _P, _P),
    "im_cuda_paged_reorder": (_P, _P, _P, _I, _P, _L, _P, _P),
    "im_cuda_beam_select_scratch_bytes": (_P, _I, _I, _I, _I),
    "im_cuda_beam_select": (_P, _P, _I, _L, _I, _I, _I, _P, _P, _I, _I, _P, _P, _P, _P, _Z, _P),
}


def use(path: str) -> None:
    """Names the library file to load, before the first call (build.ensure() returns it)."""
    global LIB_PATH
    if _lib is not None and path != LIB_PATH:
        raise CudaSysError(-7, f"{LIB_PATH} is already loaded")
    LIB_PATH = path


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise CudaSysError(-8, f"{LIB_PATH} not built: run `python -m ironmill_b200.build`")
        _lib = C.CDLL(LIB_PATH)
        _lib.im_cuda_last_error.restype = C.c_char_p
        for name in _VOIDP_RESTYPE:
            if hasattr(_lib, name):
                getattr(_lib, name).restype = C.c_void_p
        for name in _SIZE_RESTYPE:
            if hasattr(_lib, name):
                getattr(_lib, name).restype = C.c_size_t
        for name, types in _ARGTYPES.items():
            if hasattr(_lib, name):
                getattr(_lib, name).argtypes = types
        for name in _VOID_RESTYPE:
            if hasattr(_lib, name):
                getattr(_lib, name).restype = None
    return _lib


# Arguments that a call takes in a struct (im_paged_append_args and so on, include/ironmill_cuda.h): packing them is a fraction of what ctypes takes to convert as many
# arguments one by one. NULL is 0.
APPEND_ARGS = struct.Struct("11P4q9if")
PREFIX_ARGS = struct.Struct("5PN2q6if4x2P3i4x")
WEIGHTS_ARGS = struct.Struct("5PN2q6if4xP2qi4x")
EVICT_ARGS = struct.Struct("3P6q2i")


class PagedKvStruct(C.Structure):
    """im_paged_kv of include/ironmill_cuda.h."""
    _fields_ = [("k_dev", _P), ("v_dev", _P), ("layer_stride", _L), ("page_stride", _L), ("num_layers", _I), ("num_pages", _I), ("num_kv_heads", _I),
                ("page_size", _I), ("head_dim", _I), ("dtype", _I), ("num_seqs", _I), ("page_table_dev", _P), ("table_width", _I), ("table_stride", _L),
                ("seq_len_dev", _P)]


def last_error() -> str:
    return lib().im_cuda_last_error().decode("utf-8", "replace")


def check(rc: int) -> None:
    if rc != IM_OK:
        raise CudaSysError(rc, last_error())


def vp(x) -> C.c_void_p:
    """Device or host pointer argument from an int address, a torch tensor or a numpy array."""
    if x is None:
        return C.c_void_p(None)
    if isinstance(x, int):
        return C.c_void_p(x)
    if hasattr(x, "data_ptr"):
        return C.c_void_p(x.data_ptr())
    if hasattr(x, "ctypes"):
        return C.c_void_p(x.ctypes.data)
    raise TypeError(type(x))
