"""ctypes binding of libw8a8.so (the C ABI declared in include/w8a8.h).

The library is built in-tree by `python -m optimized_rocwmma_samples_amd.build`
(or `__graft_entry__.build()`).  Loading fails loudly when it is missing: there
is no CPU or PyTorch fallback for any operation of this package.
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libw8a8.so"

SUCCESS = 0
ERROR_INVALID_VALUE = 1
ERROR_NOT_SUPPORTED = 801

LAYOUT_A_ROW_B_NK = 0
LAYOUT_A_COL_B_KN = 1

OUT_I32 = 0
OUT_F16 = 1

STREAMK_WAIT_EXPIRED = 1

PLAN_MOE_QUANT = 0  # w8a8_debug_plan kinds
PLAN_GEMM = 1
PLAN_GEMM_PACKED = 2
PLAN_MOE_GEMM = 3
PLAN_GEMM_ANY = 4
PLAN_NORM_ANY = 5
PLAN_MOE_REQUANT = 6
PLAN_GROUPED = 7

GROUPED_INLINE_GROUPS = 48  # W8A8_GROUPED_INLINE_GROUPS
MOE_DECODE_MAX_TOKENS = 16  # W8A8_MOE_DECODE_MAX_TOKENS

FOLD_MULTIPLY = 0
FOLD_DIVIDE = 1

_u32 = ctypes.c_uint32
_i32 = ctypes.c_int
_f32 = ctypes.c_float
_ptr = ctypes.c_void_p
_size = ctypes.c_size_t
_u64 = ctypes.c_uint64


class GroupDesc(ctypes.Structure):
    """w8a8_group_desc (include/w8a8.h)."""
    _fields_ = [("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("c", ctypes.c_void_p),
                ("scale_a", ctypes.c_void_p), ("scale_b", ctypes.c_void_p),
                ("m", ctypes.c_uint32), ("n", ctypes.c_uint32), ("k", ctypes.c_uint32),
                ("lda", ctypes.c_uint32), ("ldb", ctypes.c_uint32), ("ldc", ctypes.c_uint32),
                ("tensor_scale_a", ctypes.c_float), ("tensor_scale_b", ctypes.c_float)]


class Kv4Cache(ctypes.Structure):
    """w8a8_kv4_cache (include/w8a8.h)."""
    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("k_scales", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("pages", ctypes.c_uint32), ("page_size", ctypes.c_uint32),
                ("kv_heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("group", ctypes.c_uint32)]


# name -> (restype, argtypes); mirrors include/w8a8.h
SIGNATURES: dict[str, tuple[object, list[object]]] = {
    "w8a8_version": (ctypes.c_char_p, []),
    "w8a8_last_error": (ctypes.c_char_p, []),
    "w8a8_smoothquant": (_i32, [_ptr, _ptr, _ptr, _ptr, _u32, _u32, _f32, _u32, _u32, _ptr]),
    "w8a8_moe_smoothquant": (_i32, [_ptr, _ptr, _ptr, _ptr, _ptr, _u32, _u32, _u32, _u32, _f32,
                                    _ptr, _u32, _ptr]),
    "w8a8_add_rmsnorm_smoothquant": (_i32, [_ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _u32,
                                            _u32, _f32, _f32, _u32, _u32, _u32, _ptr]),
    "w8a8_quantize_weights": (_i32, [_ptr, _u32, _u32, _u32, _ptr, _i32, _f32, _ptr, _u32, _i32,
                                     _size, _ptr, _ptr]),
    "w8a8_gemm_workspace_size": (_size, [_u32, _u32, _u32, _i32]),
    "w8a8_gemm": (_i32, [_u32, _u32, _u32, _ptr, _ptr, _ptr, _u32, _u32, _u32, _ptr, _ptr, _f32,
                         _f32, _i32, _i32, _ptr, _size, _ptr]),
    "w8a8_gemm_noalloc": (_i32, [_u32, _u32, _u32, _ptr, _ptr, _ptr, _u32, _u32, _u32, _ptr, _ptr,
                                 _f32, _f32, _i32, _i32, _ptr]),
    "w8a8_gemm_streamk_workspace_size": (_size, [_u32, _u32, _u32, _u32]),
    "w8a8_gemm_streamk": (_i32, [_u32, _u32, _u32, _ptr, _ptr, _ptr, _u32, _u32, _u32, _ptr, _ptr,
                                 _f32, _f32, _i32, _u32, _ptr, _size, _ptr]),
    "w8a8_gemm_streamk_blocks": (_u32, [_u32, _u32, _u32, _u32]),
    "w8a8_gemm_streamk_status": (_i32, [ctypes.POINTER(ctypes.c_uint32), _i32]),
    "w8a8_debug_streamk_wait": (_i32, [_u32, _u32]),
    "w8a8_debug_plan": (_i32, [_i32, ctypes.POINTER(ctypes.c_uint32),
                               ctypes.POINTER(ctypes.c_uint32)]),
    "w8a8_fused_sq_gemm": (_i32, [_ptr, _ptr, _ptr, _ptr, _ptr, _u32, _u32, _u32, _u32, _u32,
                                  _u32, _ptr, _ptr, _ptr, _size, _ptr]),
    "w8a8_pack_weights_size": (_size, [_u32, _u32]),
    "w8a8_pack_weights": (_i32, [_ptr, _u32, _u32, _u32, _ptr, _size, _ptr]),
    "w8a8_gemm_packed_workspace_size": (_size, [_u32, _u32, _u32]),
    "w8a8_gemm_packed": (_i32, [_u32, _u32, _u32, _ptr, _ptr, _ptr, _u32, _u32, _ptr, _ptr, _f32,
                                _f32, _i32, _ptr, _size, _ptr]),
    "w8a8_fused_sq_gemm_packed": (_i32, [_ptr, _ptr, _ptr, _ptr, _ptr, _u32, _u32, _u32, _u32,
                                         _u32, _ptr, _ptr, _ptr, _size, _ptr]),
    "w8a8_grouped_gemm_workspace_size": (_size, [_u32]),
    "w8a8_grouped_gemm": (_i32, [ctypes.POINTER(GroupDesc), _u32, _i32, _ptr, _size, _ptr]),
    "w8a8_topk_softmax": (_i32, [_ptr, _i32, _ptr, _ptr, _u32, _u32, _u32, _ptr]),
    "w8a8_moe_sort_capacity": (_size, [_u32, _u32, _u32, _u32]),
    "w8a8_moe_sort_workspace_size": (_size, [_u32, _u32, _u32]),
    "w8a8_moe_sort": (_i32, [_ptr, _u32, _u32, _u32, _u32, _ptr, _ptr, _ptr, _ptr, _u32, _ptr,
                             _ptr, _size, _ptr]),
    "w8a8_moe_gemm_workspace_size": (_size, [_u32, _u32, _u32, _u32]),
    "w8a8_moe_gemm": (_i32, [_u32, _u32, _u32, _u32, _ptr, _u32, _ptr, _u32, _u64, _ptr, _u32,
                             _ptr, _ptr, _f32, _f32, _ptr, _ptr, _i32, _ptr, _size, _ptr]),
    "w8a8_moe_silu_mul_quant": (_i32, [_ptr, _u32, _ptr, _ptr, _ptr, _u32, _u32, _u32, _ptr, _u32,
                                       _ptr, _f32, _ptr]),
    "w8a8_moe_interleave_gate_up": (_i32, [_ptr, _ptr, _u32, _u32, _u32, _u32, _ptr, _ptr, _ptr]),
    "w8a8_moe_gate_up_silu_workspace_size": (_size, [_u32, _u32]),
    "w8a8_moe_gate_up_silu": (_i32, [_u32, _u32, _u32, _u32, _ptr, _u32, _ptr, _ptr, _ptr, _f32,
                                     _f32, _ptr, _ptr, _ptr, _ptr, _u32, _ptr, _f32, _ptr, _size,
                                     _ptr]),
    "w8a8_moe_combine": (_i32, [_ptr, _u32, _u32, _ptr, _ptr, _u32, _u32, _u32, _ptr, _u32,
                                _ptr]),
    "w8a8_moe_ffn_decode_workspace_size": (_size, [_u32, _u32, _u32, _u32]),
    "w8a8_moe_ffn_decode": (_i32, [_ptr, _ptr, _i32, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr, _ptr,
                                   _u32, _u32, _u32, _u32, _u32, _f32, _u32, _u32, _ptr, _size,
                                   _ptr]),
    "w8a8_attention": (_i32, [_ptr, _ptr, _ptr, _ptr, _ptr, _u32, _u32, _u32, _u32, _u32, _u32,
                              _u32, _u32, _u32, _f32, _ptr]),
    "w8a8_kv4_store": (_i32, [_ptr, _ptr, _ptr, _u32, _u32, _u32, ctypes.POINTER(Kv4Cache),
                              _ptr]),
    "w8a8_kv4_load": (_i32, [_ptr, _ptr, _ptr, _u32, _u32, _u32, ctypes.POINTER(Kv4Cache), _ptr]),
    "w8a8_attention_kv4_workspace_size": (_size, [_u32, _u32, _u32, _u32, _u32]),
    "w8a8_attention_kv4": (_i32, [_ptr, ctypes.POINTER(Kv4Cache), _ptr, _u32, _u32, _ptr, _ptr,
                                  _u32, _u32, _u32, _u32, _f32, _ptr, _size, _ptr]),
}


class W8A8Error(RuntimeError):
    """A C-ABI call returned a non-zero status."""

    def __init__(self, fn: str, code: int, message: str):
        super().__init__(f"{fn} failed with status {code}: {message}")
        self.fn = fn
        self.code = code
        self.message = message


def _bind_hip_runtime() -> None:
    """Make libw8a8.so share the HIP runtime of the PyTorch build in use.

    PyTorch-ROCm ships its own libamdhip64.so (SONAME libamdhip64.so.7, but its
    own libraries NEED the unversioned name).  If libw8a8.so were loaded first,
    its libamdhip64.so.7 would resolve to /opt/rocm and torch would then load a
    second HIP + HSA runtime into the process: kernels launched through one
    runtime are not ordered against copies issued through the other, and two
    HSA runtimes driving one device crash.  Importing torch first lets the
    dynamic loader satisfy libamdhip64.so.7 with torch's already-loaded copy.
    """
    try:
        import torch  # noqa: F401
    except ImportError:  # C++-only users: /opt/rocm's runtime is the only one
        pass


def loaded_hip_runtimes() -> list[str]:
    """Paths of every libamdhip64 mapped into this process (should be one)."""
    with open("/proc/self/maps") as f:
        return sorted({l.split()[-1] for l in f if "libamdhip64" in l})


_lock = threading.Lock()
_lib: ctypes.CDLL | None = None


def load(path: str | Path | None = None) -> ctypes.CDLL:
    """Load libw8a8.so once and attach the C signatures."""
    global _lib
    with _lock:
        if _lib is not None and path is None:
            return _lib
        p = Path(path) if path is not None else LIB_PATH
        if not p.exists():
            raise RuntimeError(
                f"libw8a8.so not found at {p}; build it with "
                "`python -m optimized_rocwmma_samples_amd.build` (no fallback exists)")
        _bind_hip_runtime()
        lib = ctypes.CDLL(str(p))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        if path is None:
            _lib = lib
        return lib


def check(fn: str, status: int) -> None:
    if status != SUCCESS:
        msg = load().w8a8_last_error().decode(errors="replace")
        raise W8A8Error(fn, status, msg)


_calls: dict[str, object] = {}  # bound entry points of the loaded library, by name


def call(name: str, *args) -> None:
    """Call a status-returning entry point and raise W8A8Error on failure."""
    fn = _calls.get(name)
    if fn is None:
        fn = _calls[name] = getattr(load(), name)
    status = fn(*args)
    if status != SUCCESS:
        check(name, status)
