"""ctypes view of the C ABI in ``include/fa_paged_sm100.h`` (the paged key/value cache group).

The torch operators (``csrc/fa_paged_bindings.cpp``) call the same entry points from C++; tests call them
from here to check the ABI itself.  When the shared library is missing, loading raises.
"""
from __future__ import annotations

import ctypes
import os

from . import build as _build

ABI_VERSION = 1
FP16, BF16 = 0, 1
MAX_REQUESTS = 16384

EXPORTS = [
    "fa_paged_extend_sm100",
    "fa_paged_shrink_sm100",
    "fa_rotary_sm100",
    "fa_paged_append_sm100",
    "fa_paged_attention_sm100_workspace_bytes",
    "fa_paged_attention_sm100",
    "fa_paged_sm100_abi_version",
    "fa_paged_sm100_launch_count",
    "fa_paged_sm100_strerror",
]

_u32, _i32, _i64, _f32, _p = ctypes.c_uint32, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p


class PagedCacheView(ctypes.Structure):
    _fields_ = [("k", _p), ("v", _p)] + [(n, _i64) for n in (
        "k_page_stride", "k_head_stride", "k_row_stride", "v_page_stride", "v_head_stride", "v_row_stride")] + [
        (n, _i32) for n in ("num_pages", "heads_k", "page_size", "head_dim")]


class ExtendArgs(ctypes.Structure):
    _fields_ = [("struct_size", _u32), ("device", _i32), ("block_table", _p), ("table_stride", _i64)] + [
        (n, _p) for n in ("lens", "new_lens", "free_pages", "free_head", "lens_out", "head_out", "slots", "positions",
                          "cu")] + [
        (n, _i32) for n in ("batch", "table_width", "page_size", "num_free_pages")] + [("num_tokens", _i64)]


class ShrinkArgs(ctypes.Structure):
    _fields_ = [("struct_size", _u32), ("device", _i32), ("block_table", _p), ("table_stride", _i64)] + [
        (n, _p) for n in ("lens", "keep_lens", "free_pages", "free_head")] + [
        (n, _i32) for n in ("batch", "table_width", "page_size", "num_free_pages")]


class RotarySpec(ctypes.Structure):
    _fields_ = [("freqs", _p), ("positions", _p), ("positions_64", _i32), ("rot_dim", _i32), ("interleaved", _i32),
                ("adjoint", _i32), ("mscale", _f32), ("reserved", _i32)]


class RotaryArgs(ctypes.Structure):
    _fields_ = [("struct_size", _u32), ("device", _i32)] + [(n, _p) for n in ("q", "k", "q_out", "k_out")] + [
        (n, _i64) for n in ("q_batch_stride", "q_head_stride", "q_row_stride", "k_batch_stride", "k_head_stride",
                            "k_row_stride", "position_batch_stride")] + [("rotary", RotarySpec)] + [
        (n, _i32) for n in ("batch", "heads", "heads_k", "seqlen", "head_dim", "dtype")]


class AppendArgs(ctypes.Structure):
    _fields_ = [("struct_size", _u32), ("device", _i32)] + [(n, _p) for n in ("q", "k", "v", "q_out", "slots")] + [
        (n, _i64) for n in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride", "v_token_stride",
                            "v_head_stride")] + [("cache", PagedCacheView), ("rotary", RotarySpec),
                                                 ("num_tokens", _i64)] + [
        (n, _i32) for n in ("heads", "dtype", "slots_64", "reserved")]


class AttentionArgs(ctypes.Structure):
    _fields_ = [("struct_size", _u32), ("device", _i32)] + [
        (n, _p) for n in ("q", "out", "lse", "block_table", "lens", "slopes")] + [
        (n, _i64) for n in ("q_batch_stride", "q_head_stride", "table_stride")] + [("cache", PagedCacheView)] + [
        (n, _i32) for n in ("batch", "heads", "table_width", "window")] + [("scale", _f32), ("softcap", _f32)] + [
        (n, _i32) for n in ("dtype", "reserved")]


class PagedError(RuntimeError):
    def __init__(self, code: int, text: str):
        super().__init__(f"fa_paged_sm100: {text} ({code})")
        self.code = code


_lib = None


def load():
    """dlopen the C-ABI library and declare its prototypes.  Raises when absent."""
    global _lib
    if _lib is not None:
        return _lib
    path = _build.PAGED_CABI_SO
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} is not built; run `python -m custom_ops_b200.build` (needs nvcc)")
    lib = ctypes.CDLL(path)
    P = ctypes.POINTER
    lib.fa_paged_extend_sm100.argtypes = [P(ExtendArgs), _p]
    lib.fa_paged_shrink_sm100.argtypes = [P(ShrinkArgs), _p]
    lib.fa_rotary_sm100.argtypes = [P(RotaryArgs), _p]
    lib.fa_paged_append_sm100.argtypes = [P(AppendArgs), _p]
    lib.fa_paged_attention_sm100_workspace_bytes.argtypes = [P(AttentionArgs), P(ctypes.c_size_t)]
    lib.fa_paged_attention_sm100.argtypes = [P(AttentionArgs), _p, ctypes.c_size_t, _p]
    lib.fa_paged_sm100_launch_count.argtypes = [P(ctypes.c_uint64)]
    lib.fa_paged_sm100_strerror.restype = ctypes.c_char_p
    lib.fa_paged_sm100_strerror.argtypes = [ctypes.c_int]
    if lib.fa_paged_sm100_abi_version() != ABI_VERSION:
        raise RuntimeError("libfa_paged_sm100.so was built from a different ABI version")
    _lib = lib
    return lib


def check(code: int):
    if code != 0:
        raise PagedError(code, load().fa_paged_sm100_strerror(code).decode())


def workspace_bytes(args: AttentionArgs) -> int:
    n = ctypes.c_size_t(0)
    check(load().fa_paged_attention_sm100_workspace_bytes(ctypes.byref(args), ctypes.byref(n)))
    return int(n.value)


def launch_count() -> int:
    """Kernels launched by the library in this process so far."""
    n = ctypes.c_uint64(0)
    check(load().fa_paged_sm100_launch_count(ctypes.byref(n)))
    return int(n.value)
