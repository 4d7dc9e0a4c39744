"""lvb — Python host mirror of the LavaB200 Julia package, over liblvb's C ABI.

The Julia package (``lava.jl_b200/LavaB200``) is the drop-in for Lava.jl users; this module
exposes the same entry points to Python so the parity tests and the benchmark drive the
library exactly the way the Julia host does (``ccall`` ≙ ``ctypes``):

* capability vocabulary — ``MatrixShape``, ``DeviceCaps``, ``caps``, ``matrix_shapes``,
  ``supports``, ``bestshape``, ``wggranularity`` (Lava ``src/vocabulary/matrix.jl:88-172``,
  ``src/vocabulary/caps.jl:54-169``);
* ``gemm(C, A, B)`` — Lava's coopmat GEMM (``gemm!`` in Julia): ``C = A·B`` with the
  accumulation type of ``C``'s pair, layouts read from the tensors' strides (row-major
  ≙ ``Val(true)``, ``src/vocabulary/coopmat.jl:124-161``);
* ``attention(O, Q, K, V; causal, scale)`` — the flash-attention forward (``attention!``);
* ``rope(Qo, Q, pos, freqs; ...)`` — rotation of queries and keys by position, and its gradient;
* ``kv_append(...)`` and ``attention_paged(...)`` — new tokens into a paged KV cache, and the
  attention of ragged batches over it, with a prefix that all sequences share;
* ``device_status()`` — the exception-flag check Lava's host does after a sync
  (``src/compiler/entry_wrapper.jl:199-216``).

Errors are raised as ``LavaError(operation, message, suggestion)`` like Lava's
(``src/runtime/errors.jl:4-24``). There is no fallback: if ``liblvb.so`` is missing the
import fails, and a call on a machine without a B200 raises.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass, field
from pathlib import Path
from typing import Optional

_HERE = Path(__file__).resolve().parent
LIB_PATH = Path(os.environ.get("LVB_LIBRARY", _HERE.parent / "lib" / "liblvb.so"))

# ---- status / dtype enums (include/lvb.h) -------------------------------------------
LVB_OK, LVB_ERR_INVALID_ARG, LVB_ERR_UNSUPPORTED, LVB_ERR_CUDA = 0, 1, 2, 3
LVB_ERR_TIMEOUT, LVB_ERR_NCCL, LVB_ERR_NO_DEVICE = 4, 5, 6
F16, BF16, F32, I8, U8, I32, U32 = range(7)
ACT_NONE, ACT_RELU, ACT_GELU_TANH, ACT_GELU_ERF, ACT_SILU = range(5)
CLAMP_UNDEFINED, CLAMP_CONSTANT, CLAMP_TO_EDGE = range(3)
ACTIVATIONS = {None: ACT_NONE, "none": ACT_NONE, "relu": ACT_RELU, "gelu": ACT_GELU_TANH,
               "gelu_tanh": ACT_GELU_TANH, "gelu_erf": ACT_GELU_ERF, "silu": ACT_SILU}
BIAS_PER_ROW, BIAS_PER_COL = 0, 1
SUBGROUP_SCOPE, WORKGROUP_SCOPE = 0, 1
DTYPE_NAMES = {F16: "Float16", BF16: "BFloat16", F32: "Float32", I8: "Int8", U8: "UInt8",
               I32: "Int32", U32: "UInt32"}
DTYPE_SIZES = {F16: 2, BF16: 2, F32: 4, I8: 1, U8: 1, I32: 4, U32: 4}

# Symbols include/lvb.h declares; the CPU tests check the library exports each one.
EXPORTS = [
    "lvb_caps_sm100", "lvb_caps", "lvb_matrix_shapes", "lvb_bestshape",
    "lvb_gemm_check", "lvb_gemm_plan_for", "lvb_gemm", "lvb_gemm_noalloc",
    "lvb_gemm_noalloc_status", "lvb_gemm_noalloc_selftest_wait_timeout",
    "lvb_gemm_ex_check", "lvb_gemm_ex", "lvb_pe_program_check",
    "lvb_attention_check", "lvb_attention_plan_for", "lvb_attention_fwd",
    "lvb_rope_check", "lvb_rope", "lvb_kv_append_check", "lvb_kv_append",
    "lvb_attention_paged_check", "lvb_attention_paged_plan_for", "lvb_attention_paged",
    "lvb_abi_version", "lvb_last_error", "lvb_status_string", "lvb_device_count",
    "lvb_set_device", "lvb_malloc", "lvb_free", "lvb_memcpy_htod", "lvb_memcpy_dtoh",
    "lvb_stream_create", "lvb_stream_destroy", "lvb_stream_synchronize",
    "lvb_device_status", "lvb_set_wait_timeout_ms", "lvb_shard_range",
    "lvb_selftest_wait_timeout",
    "lvb_comm_unique_id", "lvb_comm_init", "lvb_comm_destroy", "lvb_comm_size", "lvb_allgather",
]


class LavaError(RuntimeError):
    """``LavaError(operation, message, suggestion)`` plus the lvb status code."""

    def __init__(self, status: int, text: str):
        self.status = status
        op, _, rest = text.partition(": ")
        msg, _, hint = rest.partition(" (")
        self.operation = op
        self.message = msg
        self.suggestion = hint[:-1] if hint.endswith(")") else hint
        super().__init__(f"[{STATUS_NAMES.get(status, status)}] {text}")


STATUS_NAMES = {0: "LVB_OK", 1: "LVB_ERR_INVALID_ARG", 2: "LVB_ERR_UNSUPPORTED",
                3: "LVB_ERR_CUDA", 4: "LVB_ERR_TIMEOUT", 5: "LVB_ERR_NCCL",
                6: "LVB_ERR_NO_DEVICE"}


# ---- C structs ------------------------------------------------------------------------
class lvb_matrix_shape(C.Structure):
    _fields_ = [("ab", C.c_int32), ("acc", C.c_int32), ("M", C.c_int32), ("N", C.c_int32),
                ("K", C.c_int32), ("scope", C.c_int32)]


class lvb_device_caps(C.Structure):
    _fields_ = [("coopmat", C.c_int32), ("tile", C.c_int32), ("subgroup", C.c_int32),
                ("coopmatsubgroup", C.c_int32), ("sharedbudget", C.c_int64),
                ("workgrouplimit", C.c_int32), ("cores", C.c_int32), ("warps", C.c_int32),
                ("n_wggran", C.c_int32), ("wggran", (C.c_int32 * 4) * 8),
                ("n_shapes", C.c_int32), ("cc_major", C.c_int32), ("cc_minor", C.c_int32)]


class lvb_gemm_desc(C.Structure):
    _fields_ = [("a_type", C.c_int32), ("b_type", C.c_int32), ("c_type", C.c_int32),
                ("a_rowmajor", C.c_int32), ("b_rowmajor", C.c_int32), ("c_rowmajor", C.c_int32),
                ("M", C.c_int64), ("N", C.c_int64), ("K", C.c_int64),
                ("lda", C.c_int64), ("ldb", C.c_int64), ("ldc", C.c_int64)]


class lvb_gemm_plan(C.Structure):
    _fields_ = [("swap_ab", C.c_int32), ("tile_m", C.c_int32), ("tile_n", C.c_int32),
                ("tile_k", C.c_int32), ("stages", C.c_int32), ("tiles", C.c_int32),
                ("ctas", C.c_int32), ("smem_bytes", C.c_int32), ("tmem_cols", C.c_int32),
                ("instr_m", C.c_int32), ("instr_n", C.c_int32), ("instr_k", C.c_int32),
                ("repack_a", C.c_int32), ("repack_b", C.c_int32), ("cta_pair", C.c_int32),
                ("a_mnmajor", C.c_int32), ("b_mnmajor", C.c_int32), ("gemv", C.c_int32),
                ("gemv_ksplit", C.c_int32), ("launches", C.c_int32)]


class lvb_attn_plan(C.Structure):
    _fields_ = [("kernel", C.c_int32), ("splits", C.c_int32), ("ctas", C.c_int32),
                ("launches", C.c_int32)]


class lvb_epilogue(C.Structure):
    _fields_ = [("bias", C.c_void_p), ("residual", C.c_void_p), ("ldr", C.c_int64),
                ("bias_type", C.c_int32), ("bias_axis", C.c_int32),
                ("residual_type", C.c_int32), ("activation", C.c_int32),
                ("mul", C.c_void_p), ("ldm", C.c_int64), ("mul_type", C.c_int32),
                ("extra_type", C.c_int32), ("extra", C.c_void_p), ("lde", C.c_int64),
                ("program", C.c_void_p), ("k_pad", C.c_int64),
                ("a_clamp", C.c_int32), ("b_clamp", C.c_int32),
                ("a_clamp_value", C.c_double), ("b_clamp_value", C.c_double)]


class lvb_attn_desc(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("causal", C.c_int32),
                ("batch", C.c_int64), ("heads_q", C.c_int64), ("heads_kv", C.c_int64),
                ("seq_q", C.c_int64), ("seq_kv", C.c_int64), ("head_dim", C.c_int64),
                ("scale", C.c_float), ("reserved", C.c_int32),
                ("q_stride", C.c_int64 * 3), ("k_stride", C.c_int64 * 3),
                ("v_stride", C.c_int64 * 3), ("o_stride", C.c_int64 * 3)]


class lvb_rotation(C.Structure):
    _fields_ = [("pairs", C.c_int32), ("layout", C.c_int32), ("n_axes", C.c_int32),
                ("inverse", C.c_int32), ("sections", C.c_int32 * 4)]


class lvb_rope_desc(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("reserved", C.c_int32),
                ("batch", C.c_int64), ("heads_q", C.c_int64), ("heads_kv", C.c_int64),
                ("seq", C.c_int64), ("head_dim", C.c_int64),
                ("q_stride", C.c_int64 * 3), ("k_stride", C.c_int64 * 3),
                ("qo_stride", C.c_int64 * 3), ("ko_stride", C.c_int64 * 3),
                ("pos_stride", C.c_int64 * 3), ("rot", lvb_rotation)]


class lvb_paged_desc(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("causal", C.c_int32),
                ("batch", C.c_int64), ("heads_q", C.c_int64), ("heads_kv", C.c_int64),
                ("head_dim", C.c_int64), ("tokens", C.c_int64), ("max_q", C.c_int64),
                ("page_size", C.c_int64), ("num_pages", C.c_int64), ("table_width", C.c_int64),
                ("table_stride", C.c_int64), ("prefix_len", C.c_int64),
                ("kc_stride", C.c_int64 * 3), ("vc_stride", C.c_int64 * 3),
                ("q_stride", C.c_int64 * 2), ("o_stride", C.c_int64 * 2),
                ("scale", C.c_float), ("reserved", C.c_int32)]


class lvb_append_desc(C.Structure):
    _fields_ = [("paged", lvb_paged_desc), ("k_stride", C.c_int64 * 2),
                ("v_stride", C.c_int64 * 2), ("pos_stride", C.c_int64), ("rot", lvb_rotation)]


class lvb_paged_plan(C.Structure):
    _fields_ = [("kernel", C.c_int32), ("splits", C.c_int32), ("prefix_splits", C.c_int32),
                ("cluster", C.c_int32), ("launches", C.c_int32), ("reserved", C.c_int32),
                ("workspace_bytes", C.c_int64)]


class lvb_comm_id(C.Structure):
    _fields_ = [("bytes", C.c_char * 128)]


def _load() -> C.CDLL:
    if not LIB_PATH.exists():
        raise ImportError(f"liblvb.so not built at {LIB_PATH}; run python lava.jl_b200/build.py")
    lib = C.CDLL(str(LIB_PATH))
    P = C.c_void_p
    sig = {
        "lvb_caps_sm100": ([C.POINTER(lvb_device_caps)], C.c_int),
        "lvb_caps": ([C.c_int, C.POINTER(lvb_device_caps)], C.c_int),
        "lvb_matrix_shapes": ([C.POINTER(lvb_matrix_shape), C.c_int32, C.POINTER(C.c_int32)], C.c_int),
        "lvb_bestshape": ([C.c_int32, C.c_int32, C.c_int32, C.POINTER(lvb_matrix_shape)], C.c_int),
        "lvb_gemm_check": ([C.POINTER(lvb_gemm_desc)], C.c_int),
        "lvb_gemm_plan_for": ([C.POINTER(lvb_gemm_desc), C.c_int32, C.POINTER(lvb_gemm_plan)], C.c_int),
        "lvb_gemm": ([C.POINTER(lvb_gemm_desc), P, P, P, P], C.c_int),
        "lvb_gemm_noalloc": ([C.POINTER(lvb_gemm_desc), P, P, P, P], C.c_int),
        "lvb_gemm_noalloc_status": ([P, C.POINTER(C.c_int32), C.POINTER(C.c_int32),
                                     C.POINTER(C.c_int32)], C.c_int),
        "lvb_gemm_noalloc_selftest_wait_timeout": ([C.c_int32, P], C.c_int),
        "lvb_gemm_ex_check": ([C.POINTER(lvb_gemm_desc), C.POINTER(lvb_epilogue)], C.c_int),
        "lvb_pe_program_check": ([P], C.c_int),
        "lvb_gemm_ex": ([C.POINTER(lvb_gemm_desc), C.POINTER(lvb_epilogue), P, P, P, P], C.c_int),
        "lvb_attention_check": ([C.POINTER(lvb_attn_desc)], C.c_int),
        "lvb_attention_fwd": ([C.POINTER(lvb_attn_desc), P, P, P, P, P, P], C.c_int),
        "lvb_attention_plan_for": ([C.POINTER(lvb_attn_desc), C.c_int32, C.POINTER(lvb_attn_plan)], C.c_int),
        "lvb_rope_check": ([C.POINTER(lvb_rope_desc)], C.c_int),
        "lvb_rope": ([C.POINTER(lvb_rope_desc)] + [P] * 7, C.c_int),
        "lvb_kv_append_check": ([C.POINTER(lvb_append_desc)], C.c_int),
        "lvb_kv_append": ([C.POINTER(lvb_append_desc)] + [P] * 12, C.c_int),
        "lvb_attention_paged_check": ([C.POINTER(lvb_paged_desc)], C.c_int),
        "lvb_attention_paged_plan_for": ([C.POINTER(lvb_paged_desc), C.c_int32,
                                          C.POINTER(lvb_paged_plan)], C.c_int),
        "lvb_attention_paged": ([C.POINTER(lvb_paged_desc)] + [P] * 10, C.c_int),
        "lvb_abi_version": ([], C.c_int),
        "lvb_last_error": ([], C.c_char_p),
        "lvb_status_string": ([C.c_int], C.c_char_p),
        "lvb_device_count": ([C.POINTER(C.c_int32)], C.c_int),
        "lvb_set_device": ([C.c_int], C.c_int),
        "lvb_malloc": ([C.POINTER(P), C.c_size_t], C.c_int),
        "lvb_free": ([P], C.c_int),
        "lvb_memcpy_htod": ([P, P, C.c_size_t, P], C.c_int),
        "lvb_memcpy_dtoh": ([P, P, C.c_size_t, P], C.c_int),
        "lvb_stream_create": ([C.POINTER(P)], C.c_int),
        "lvb_stream_destroy": ([P], C.c_int),
        "lvb_stream_synchronize": ([P], C.c_int),
        "lvb_device_status": ([P, C.POINTER(C.c_int32), C.POINTER(C.c_int32), C.POINTER(C.c_int32)], C.c_int),
        "lvb_set_wait_timeout_ms": ([C.c_int64], C.c_int),
        "lvb_shard_range": ([C.c_int64, C.c_int32, C.c_int32, C.c_int64, C.POINTER(C.c_int64),
                             C.POINTER(C.c_int64)], C.c_int),
        "lvb_selftest_wait_timeout": ([C.c_int32, P], C.c_int),
        "lvb_comm_unique_id": ([C.POINTER(lvb_comm_id)], C.c_int),
        "lvb_comm_init": ([C.POINTER(P), C.POINTER(lvb_comm_id), C.c_int32, C.c_int32], C.c_int),
        "lvb_comm_destroy": ([P], C.c_int),
        "lvb_comm_size": ([P, C.POINTER(C.c_int32), C.POINTER(C.c_int32)], C.c_int),
        "lvb_allgather": ([P, P, P, C.c_size_t, P], C.c_int),
    }
    for name, (args, res) in sig.items():
        f = getattr(lib, name)
        f.argtypes = args
        f.restype = res
    return lib


lib = _load()


def check(status: int) -> None:
    if status != LVB_OK:
        raise LavaError(status, lib.lvb_last_error().decode())


# ---- capability vocabulary ----------------------------------------------------------
@dataclass(frozen=True)
class MatrixShape:
    """One (M, N, K) shape for operands ``ab`` accumulating into ``acc`` (matrix.jl:88-95)."""
    ab: int
    acc: int
    M: int
    N: int
    K: int
    scope: int = SUBGROUP_SCOPE

    def __str__(self):
        sc = "SubgroupScope" if self.scope == SUBGROUP_SCOPE else "WorkgroupScope"
        return (f"MatrixShape({DTYPE_NAMES[self.ab]}->{DTYPE_NAMES[self.acc]} "
                f"{self.M}x{self.N}x{self.K} {sc})")


@dataclass
class DeviceCaps:
    """Lava's DeviceCaps record (caps.jl:54-65) as a B200 answers it."""
    coopmat: bool
    tile: int
    subgroup: int
    coopmatsubgroup: int
    sharedbudget: int
    workgrouplimit: int
    cores: int
    warps: int
    wggran: list = field(default_factory=list)
    shapes: list = field(default_factory=list)


def _shape_table() -> list[MatrixShape]:
    n = C.c_int32()
    check(lib.lvb_matrix_shapes(None, 0, C.byref(n)))
    arr = (lvb_matrix_shape * n.value)()
    check(lib.lvb_matrix_shapes(arr, n.value, C.byref(n)))
    return [MatrixShape(s.ab, s.acc, s.M, s.N, s.K, s.scope) for s in arr]


def _caps_from(c: lvb_device_caps) -> DeviceCaps:
    shapes = [s for s in _shape_table() if s.scope == SUBGROUP_SCOPE]
    wg = [tuple(c.wggran[i]) for i in range(c.n_wggran)]
    return DeviceCaps(bool(c.coopmat), c.tile, c.subgroup, c.coopmatsubgroup, c.sharedbudget,
                      c.workgrouplimit, c.cores, c.warps, wg, shapes)


def caps(device: Optional[int] = None) -> DeviceCaps:
    """``Lava.caps(backend)``: the live device's answer; ``device=None`` gives the static
    sm_100a table (no GPU needed), the form Lava's copy constructor exists for."""
    c = lvb_device_caps()
    if device is None:
        check(lib.lvb_caps_sm100(C.byref(c)))
    else:
        check(lib.lvb_caps(device, C.byref(c)))
    return _caps_from(c)


def matrix_shapes(c: Optional[DeviceCaps] = None, scope: Optional[int] = None) -> list[MatrixShape]:
    """``matrix_shapes(c)``: empty when ``c.coopmat`` is false (caps.jl:158-159). With no
    caps, the whole table including the workgroup-scope (tcgen05 tile) shapes."""
    if c is not None:
        return list(c.shapes) if c.coopmat else []
    t = _shape_table()
    return [s for s in t if scope is None or s.scope == scope]


def supports(shapes_or_caps, s: MatrixShape) -> bool:
    shapes = matrix_shapes(shapes_or_caps) if isinstance(shapes_or_caps, DeviceCaps) else shapes_or_caps
    return any(x == s for x in shapes)


def _isbetter(a: MatrixShape, b: MatrixShape) -> bool:
    sa = abs(a.M - a.N) + abs(a.N - a.K)
    sb = abs(b.M - b.N) + abs(b.N - b.K)
    if sa != sb:
        return sa < sb
    return a.M * a.N * a.K > b.M * b.N * b.K


def bestshape(shapes_or_caps, ab: int, acc: int, scope: int = SUBGROUP_SCOPE) -> Optional[MatrixShape]:
    """Squarest, then largest (matrix.jl:155-172); None where Lava returns ``nothing``."""
    shapes = matrix_shapes(shapes_or_caps) if isinstance(shapes_or_caps, DeviceCaps) else shapes_or_caps
    best = None
    for s in shapes:
        if s.ab != ab or s.acc != acc or s.scope != scope:
            continue
        if best is None or _isbetter(s, best):
            best = s
    return best


def bestshape_native(ab: int, acc: int, scope: int = SUBGROUP_SCOPE) -> Optional[MatrixShape]:
    """The library's own bestshape over its full table (C ABI lvb_bestshape)."""
    out = lvb_matrix_shape()
    st = lib.lvb_bestshape(ab, acc, scope, C.byref(out))
    if st == LVB_ERR_UNSUPPORTED:
        return None
    check(st)
    return MatrixShape(out.ab, out.acc, out.M, out.N, out.K, out.scope)


def wggranularity(c: DeviceCaps, nt: int):
    """(M, N, K) multiples of a workgroup-scope matrix at ``nt`` invocations (caps.jl:140-145)."""
    for (n, m, nn, k) in c.wggran:
        if n == nt:
            return (m, nn, k)
    return None


# ---- tensors -> descriptors -----------------------------------------------------------
def _torch():
    import torch
    return torch


def dtype_of(t) -> int:
    torch = _torch()
    m = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32, torch.int8: I8,
         torch.uint8: U8, torch.int32: I32}
    if hasattr(torch, "uint32"):
        m[torch.uint32] = U32
    if t.dtype not in m:
        raise LavaError(LVB_ERR_UNSUPPORTED, f"lvb: no component type for {t.dtype}")
    return m[t.dtype]


def _layout2d(t, name: str):
    """(rowmajor, ld) of a 2-D tensor: row-major when the column stride is 1."""
    if t.dim() != 2:
        raise LavaError(LVB_ERR_INVALID_ARG, f"lvb_gemm: {name} must be 2-D")
    r, c = t.shape
    s0, s1 = t.stride()
    if r == 0 or c == 0:            # an empty operand has no layout to read
        return 1, max(c, 1)
    if s1 == 1 and (r <= 1 or s0 >= max(c, 1)):
        return 1, max(s0, c, 1)
    if s0 == 1 and (c <= 1 or s1 >= max(r, 1)):
        return 0, max(s1, r, 1)
    raise LavaError(LVB_ERR_UNSUPPORTED, f"lvb_gemm: {name} has no unit stride "
                    "(make it contiguous or a transpose of a contiguous tensor)")


def gemm_desc(C_, A, B, c_type: Optional[int] = None) -> lvb_gemm_desc:
    M, K = A.shape
    K2, N = B.shape
    if K2 != K or tuple(C_.shape) != (M, N):
        raise LavaError(LVB_ERR_INVALID_ARG,
                        f"lvb_gemm: shapes {tuple(A.shape)} x {tuple(B.shape)} -> {tuple(C_.shape)}")
    d = lvb_gemm_desc()
    d.a_type, d.b_type = dtype_of(A), dtype_of(B)
    d.c_type = dtype_of(C_) if c_type is None else c_type
    d.a_rowmajor, d.lda = _layout2d(A, "A")
    d.b_rowmajor, d.ldb = _layout2d(B, "B")
    d.c_rowmajor, d.ldc = _layout2d(C_, "C")
    d.M, d.N, d.K = M, N, K
    return d


def _stream_ptr(stream) -> Optional[int]:
    if stream is None:
        torch = _torch()
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _cmatrix(C_, t, what):
    """(pointer, type, leading dimension) of an M×N epilogue operand read in C's layout (a
    single row or column reads the same in either, whatever strides torch gave it)."""
    if tuple(t.shape) != tuple(C_.shape):
        raise LavaError(LVB_ERR_INVALID_ARG, f"lvb_gemm_ex: {what} must have C's shape")
    crm, _ = _layout2d(C_, "C")
    r, c = t.shape
    s0, s1 = t.stride()
    if crm:
        if c > 1 and s1 != 1:
            raise LavaError(LVB_ERR_UNSUPPORTED, f"lvb_gemm_ex: {what} must have C's layout")
        ld = s0 if r > 1 else max(c, 1)
    else:
        if r > 1 and s0 != 1:
            raise LavaError(LVB_ERR_UNSUPPORTED, f"lvb_gemm_ex: {what} must have C's layout")
        ld = s1 if c > 1 else max(r, 1)
    return t.data_ptr(), dtype_of(t), ld


def _clamp(spec):
    """A clamp given as None / "undefined", "edge", or a number (the constant)."""
    if spec is None or spec == "undefined":
        return CLAMP_UNDEFINED, 0.0
    if spec == "edge":
        return CLAMP_TO_EDGE, 0.0
    if isinstance(spec, (int, float)) and not isinstance(spec, bool):
        return CLAMP_CONSTANT, float(spec)
    raise LavaError(LVB_ERR_INVALID_ARG, f"lvb_gemm_ex: clamp {spec!r}: None, 'edge' or a number")


def epilogue(C_, bias=None, bias_axis: str = "col", residual=None, activation=None, mul=None,
             program=None, extra=None, k_pad=None, a_clamp=None, b_clamp=None) -> lvb_epilogue:
    """The ``lvb_epilogue`` for ``C = f(act((A·B + bias + residual) ⊙ mul))``: ``bias`` a
    contiguous vector added per column (``bias_axis="col"``, N elements) or per row (``"row"``,
    M elements); ``residual`` and ``mul`` M×N tensors in C's layout (the residual may be C
    itself); ``program`` a ``perelement.Program`` (or a Python function, traced) with
    ``extra`` its M×N matrix operand; ``k_pad`` the padded k extent whose reads past K take
    ``a_clamp`` / ``b_clamp`` (None, ``"edge"`` or a constant). The program structure is kept
    alive on the returned value (``e._keep``) for the duration of the call."""
    e = lvb_epilogue()
    if activation not in ACTIVATIONS:
        raise LavaError(LVB_ERR_INVALID_ARG, f"lvb_gemm_ex: unknown activation {activation!r}")
    e.activation = ACTIVATIONS[activation]
    if bias is not None:
        if bias.dim() != 1 or bias.stride(0) != 1:
            raise LavaError(LVB_ERR_INVALID_ARG, "lvb_gemm_ex: bias must be a contiguous vector")
        want = C_.shape[1] if bias_axis == "col" else C_.shape[0]
        if bias.shape[0] != want:
            raise LavaError(LVB_ERR_INVALID_ARG,
                            f"lvb_gemm_ex: bias has {bias.shape[0]} elements, needs {want}")
        e.bias = bias.data_ptr()
        e.bias_type = dtype_of(bias)
        e.bias_axis = BIAS_PER_COL if bias_axis == "col" else BIAS_PER_ROW
    if residual is not None:
        e.residual, e.residual_type, e.ldr = _cmatrix(C_, residual, "residual")
    if mul is not None:
        e.mul, e.mul_type, e.ldm = _cmatrix(C_, mul, "mul")
    e._keep = None
    if program is not None:
        from .perelement import Program, program as trace
        prog = program if isinstance(program, Program) else trace(program)
        st = prog.to_struct()
        e._keep = st
        e.program = C.addressof(st)
        if extra is not None:
            e.extra, e.extra_type, e.lde = _cmatrix(C_, extra, "extra")
    elif extra is not None:
        raise LavaError(LVB_ERR_INVALID_ARG, "lvb_gemm_ex: extra without a program")
    if k_pad is not None:
        e.k_pad = int(k_pad)
        e.a_clamp, e.a_clamp_value = _clamp(a_clamp)
        e.b_clamp, e.b_clamp_value = _clamp(b_clamp)
    return e


def gemm(C_, A, B, stream=None, c_type: Optional[int] = None, bias=None, bias_axis="col",
         residual=None, activation=None, mul=None, program=None, extra=None, k_pad=None,
         a_clamp=None, b_clamp=None):
    """``gemm!(C, A, B)``: C = A·B on the GPU (torch CUDA tensors, logical shapes
    (M,K)·(K,N) -> (M,N)); enqueued on ``stream`` (default: torch's current stream).
    ``c_type`` overrides the component type read from C (e.g. U32 held in an int32
    tensor). With any of the epilogue keywords the fused epilogue runs (``lvb_gemm_ex``, see
    ``epilogue``): C = program(act((A·B + bias + residual) ⊙ mul)), the product over
    ``k_pad`` columns with the clamp modes when given."""
    d = gemm_desc(C_, A, B, c_type)
    if (bias is None and residual is None and activation in (None, "none") and mul is None
            and program is None and k_pad is None):
        check(lib.lvb_gemm(C.byref(d), A.data_ptr(), B.data_ptr(), C_.data_ptr(),
                           _stream_ptr(stream)))
        return C_
    e = epilogue(C_, bias, bias_axis, residual, activation, mul, program, extra, k_pad,
                 a_clamp, b_clamp)
    check(lib.lvb_gemm_ex(C.byref(d), C.byref(e), A.data_ptr(), B.data_ptr(), C_.data_ptr(),
                          _stream_ptr(stream)))
    return C_


class GemmCall:
    """A GEMM validated and described once, launched many times: ``g = prepare_gemm(C, A, B,
    ...)`` then ``g()`` (or ``g(stream)``) enqueues ``lvb_gemm`` / ``lvb_gemm_ex`` with the
    prepared descriptor — one foreign call per launch, for small problems whose time is the
    host's. The tensors must stay alive and keep their storage while the object is used."""

    def __init__(self, C_, A, B, c_type=None, **epi):
        self.d = gemm_desc(C_, A, B, c_type)
        self.ptrs = (A.data_ptr(), B.data_ptr(), C_.data_ptr())
        self.keep = (C_, A, B)
        active = {k: v for k, v in epi.items() if v is not None and v != "none"}
        self.e = epilogue(C_, **epi) if active else None
        self._fn = lib.lvb_gemm if self.e is None else lib.lvb_gemm_ex
        self._d = C.byref(self.d)
        self._args = ((self._d,) if self.e is None else (self._d, C.byref(self.e))) + self.ptrs
        self._default_stream = None

    def __call__(self, stream=None):
        if stream is None:
            if self._default_stream is None:
                self._default_stream = _stream_ptr(None)
            s = self._default_stream
        else:
            s = _stream_ptr(stream)
        st = self._fn(*self._args, s)
        if st:
            check(st)


def prepare_gemm(C_, A, B, c_type=None, **epi) -> GemmCall:
    """See ``GemmCall``; keywords as ``gemm``'s epilogue keywords. The default stream is
    torch's current stream at the first call."""
    return GemmCall(C_, A, B, c_type, **epi)


def gemm_plan(M, N, K, a_type=F16, c_type=F32, c_rowmajor=False, sm_count=148,
              a_rowmajor=True, b_rowmajor=False) -> lvb_gemm_plan:
    lda = max(K if a_rowmajor else M, 1)
    ldb = max(N if b_rowmajor else K, 1)
    d = lvb_gemm_desc(a_type, a_type, c_type, int(a_rowmajor), int(b_rowmajor), int(c_rowmajor),
                      M, N, K, lda, ldb, max(N if c_rowmajor else M, 1))
    p = lvb_gemm_plan()
    check(lib.lvb_gemm_plan_for(C.byref(d), sm_count, C.byref(p)))
    return p


def _strides4(t):
    if t.dim() != 4 or t.stride(3) != 1:
        raise LavaError(LVB_ERR_UNSUPPORTED, "lvb_attention_fwd: tensors are [B][H][S][D] "
                        "with D contiguous")
    return (t.stride(0), t.stride(1), t.stride(2))


def attention_desc(O, Q, K, V, causal=True, scale=None) -> lvb_attn_desc:
    Bq, Hq, Sq, D = Q.shape
    Bk, Hkv, Skv, Dk = K.shape
    if tuple(V.shape) != tuple(K.shape) or Bk != Bq or Dk != D or tuple(O.shape) != tuple(Q.shape):
        raise LavaError(LVB_ERR_INVALID_ARG, "lvb_attention_fwd: shape mismatch")
    d = lvb_attn_desc()
    d.dtype = dtype_of(Q)
    if dtype_of(K) != d.dtype or dtype_of(V) != d.dtype or dtype_of(O) != d.dtype:
        raise LavaError(LVB_ERR_UNSUPPORTED, "lvb_attention_fwd: Q, K, V, O must share a dtype")
    d.causal = int(bool(causal))
    d.batch, d.heads_q, d.heads_kv, d.seq_q, d.seq_kv, d.head_dim = Bq, Hq, Hkv, Sq, Skv, D
    d.scale = float(scale) if scale is not None else float(D) ** -0.5
    for name, t in (("q_stride", Q), ("k_stride", K), ("v_stride", V), ("o_stride", O)):
        s = _strides4(t)
        arr = getattr(d, name)
        for i in range(3):
            arr[i] = s[i]
    return d


def attention(O, Q, K, V, causal=True, scale=None, lse=None, stream=None):
    """``attention!(O, Q, K, V; causal, scale)``: flash-attention forward on the GPU.
    Q/O [B][Hq][Sq][D], K/V [B][Hkv][Skv][D]; optional fp32 ``lse`` [B][Hq][Sq]."""
    d = attention_desc(O, Q, K, V, causal, scale)
    check(lib.lvb_attention_fwd(C.byref(d), Q.data_ptr(), K.data_ptr(), V.data_ptr(),
                                O.data_ptr(), lse.data_ptr() if lse is not None else None,
                                _stream_ptr(stream)))
    return O


class AttentionCall:
    """An attention forward described once, launched many times: ``a = prepare_attention(O,
    Q, K, V, ...)`` then ``a()`` (or ``a(stream)``) — one foreign call per launch. The tensors
    must stay alive and keep their storage while the object is used."""

    def __init__(self, O, Q, K, V, causal=True, scale=None, lse=None):
        self.d = attention_desc(O, Q, K, V, causal, scale)
        self.keep = (O, Q, K, V, lse)
        self._args = (C.byref(self.d), Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(),
                      lse.data_ptr() if lse is not None else None)
        self._default_stream = None

    def __call__(self, stream=None):
        if stream is None:
            if self._default_stream is None:
                self._default_stream = _stream_ptr(None)
            s = self._default_stream
        else:
            s = _stream_ptr(stream)
        st = lib.lvb_attention_fwd(*self._args, s)
        if st:
            check(st)


def prepare_attention(O, Q, K, V, causal=True, scale=None, lse=None) -> AttentionCall:
    """See ``AttentionCall``; arguments as ``attention``'s. The default stream is torch's
    current stream at the first call."""
    return AttentionCall(O, Q, K, V, causal, scale, lse)


ATTN_FLASH, ATTN_DECODE, ATTN_EMPTY = 0, 1, 2


def attention_plan(B, Hq, Hkv, Sq, Skv, D=128, dtype=BF16, causal=True,
                   sm_count=148) -> lvb_attn_plan:
    """The kernel lvb_attention_fwd picks for these extents (host only, no GPU)."""
    d = lvb_attn_desc()
    d.dtype, d.causal = dtype, int(bool(causal))
    d.batch, d.heads_q, d.heads_kv, d.seq_q, d.seq_kv, d.head_dim = B, Hq, Hkv, Sq, Skv, D
    d.scale = float(D) ** -0.5
    p = lvb_attn_plan()
    check(lib.lvb_attention_plan_for(C.byref(d), sm_count, C.byref(p)))
    return p


# ---- position rotation, paged KV cache ---------------------------------------------------
ROPE_LAYOUTS = {"halves": 0, "pairs": 1}
PAGED_FLASH, PAGED_DECODE = 0, 1


def _refuse(op, message, status=LVB_ERR_INVALID_ARG):
    raise LavaError(status, f"{op}: {message}")


def _rows(op, name, t, extents):
    """Element strides of a tensor whose last dimension (head_dim) is contiguous; a dimension of
    extent 1 gets one that any tensor could have (torch leaves it as it was). Rows that share
    elements (an expanded tensor) are refused here: in the descriptor, strides that are all 0 stand
    for the packed layout."""
    if tuple(t.shape[:-1]) != tuple(extents):
        _refuse(op, f"{name} has shape {tuple(t.shape)}, needs {tuple(extents)} rows")
    D = t.shape[-1]
    if D > 1 and t.stride(-1) != 1:
        _refuse(op, f"{name}: head_dim must be contiguous", LVB_ERR_UNSUPPORTED)
    if any(n > 1 and t.stride(i) < D for i, n in enumerate(extents)):
        _refuse(op, f"{name}: stride below head_dim (an expanded tensor needs a copy)")
    return [t.stride(i) if n > 1 else D for i, n in enumerate(extents)]


def _list_of(op, name, t, dtype, n=None):
    """A contiguous 1-D list (int32 or float64), with at least n entries."""
    if t.dtype != dtype or t.dim() != 1 or (t.shape[0] > 1 and t.stride(0) != 1):
        _refuse(op, f"{name} must be a contiguous vector of {dtype}")
    if n is not None and t.shape[0] < n:
        _refuse(op, f"{name} has {t.shape[0]} entries, needs {n}")
    return t


def _on_current_device(op, tensors):
    """Every tensor on the current CUDA device, where the kernels run."""
    torch = _torch()
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            _refuse(op, f"{name} is not a CUDA tensor")
        if t.device.index != torch.cuda.current_device():
            _refuse(op, f"{name} is on {t.device}, the current device is "
                        f"cuda:{torch.cuda.current_device()}")


def _ptr(t):
    return C.c_void_p(t.data_ptr() if t is not None else None)


class PreparedCall:
    """A call of the library described once and made many times: ``c = prepare_...(...)``, then
    ``c()`` (torch's current stream) or ``c(stream)``: one foreign call. The tensors must stay
    alive and keep their storage while the object is used (it holds them); what they hold may
    change between calls, and a call captured into a CUDA graph reads it at the replay."""

    def __init__(self, fn, desc, pointers, keep):
        self.d = desc
        self.keep = keep
        self._fn = fn
        self._args = (C.byref(desc), *pointers)
        self._device = next(t for t in keep if t is not None).device.index

    def __call__(self, stream=None):
        c = _torch()._C
        if c._cuda_getDevice() != self._device:
            raise LavaError(LVB_ERR_INVALID_ARG, "lvb: the call's tensors are on "
                            f"cuda:{self._device}, the current device is cuda:{c._cuda_getDevice()}")
        s = c._cuda_getCurrentRawStream(self._device) if stream is None else _stream_ptr(stream)
        st = self._fn(*self._args, s)
        if st:
            check(st)


def _rotation(op, freqs, sections, layout, inverse):
    torch = _torch()
    _list_of(op, "freqs", freqs, torch.float64)
    if layout not in ROPE_LAYOUTS:
        _refuse(op, f"layout {layout!r}: 'halves' or 'pairs'")
    r = lvb_rotation()
    r.pairs = freqs.shape[0]
    r.layout = ROPE_LAYOUTS[layout]
    r.inverse = int(bool(inverse))
    sections = [r.pairs] if sections is None else [int(x) for x in sections]
    if not 1 <= len(sections) <= 4:
        _refuse(op, f"{len(sections)} sections: 1 to 4 axes")
    r.n_axes = len(sections)
    for i, x in enumerate(sections):
        r.sections[i] = x
    return r


def prepare_rope(Qo, Q, pos, freqs, Ko=None, K=None, sections=None, layout="halves",
                 inverse=False) -> PreparedCall:
    """``rope`` described once (see ``PreparedCall``)."""
    op = "lvb_rope"
    if Q.dim() != 4 or Qo.shape != Q.shape:
        _refuse(op, f"Q and Qo are [B][H][S][D] of one shape, got {tuple(Q.shape)} and {tuple(Qo.shape)}")
    if (K is None) != (Ko is None):
        _refuse(op, "K and Ko come together")
    B, Hq, S, D = Q.shape
    d = lvb_rope_desc()
    d.dtype = dtype_of(Q)
    d.batch, d.heads_q, d.seq, d.head_dim = B, Hq, S, D
    d.rot = _rotation(op, freqs, sections, layout, inverse)
    pairs = [("q_stride", "Q", Q), ("qo_stride", "Qo", Qo)]
    if K is not None:
        if K.dim() != 4 or (K.shape[0], K.shape[2], K.shape[3]) != (B, S, D) or Ko.shape != K.shape:
            _refuse(op, f"K and Ko are [B][H][S][D] as Q is, got {tuple(K.shape)} and {tuple(Ko.shape)}")
        d.heads_kv = K.shape[1]
        pairs += [("k_stride", "K", K), ("ko_stride", "Ko", Ko)]
    for field_, name, t in pairs:
        if t.dtype != Q.dtype:
            _refuse(op, "Q, K and their results must share a dtype", LVB_ERR_UNSUPPORTED)
        getattr(d, field_)[:] = _rows(op, name, t, t.shape[:3])
    if pos.dtype != _torch().int32:
        _refuse(op, "pos must be int32")
    p = pos if pos.dim() == 3 else pos.unsqueeze(0)
    if p.dim() != 3 or p.shape[0] != d.rot.n_axes or p.shape[1] not in (1, B) or p.shape[2] != S:
        _refuse(op, f"pos is [{B} or 1][{S}], or [{d.rot.n_axes}][{B} or 1][{S}] for several axes, "
                    f"got {tuple(pos.shape)}")
    d.pos_stride[:] = [p.stride(0), p.stride(1) if p.shape[1] > 1 else 0, p.stride(2)]
    check(lib.lvb_rope_check(C.byref(d)))
    _on_current_device(op, {"Qo": Qo, "Q": Q, "pos": pos, "freqs": freqs, "Ko": Ko, "K": K})
    return PreparedCall(lib.lvb_rope, d, (_ptr(Q), _ptr(K), _ptr(Qo), _ptr(Ko), _ptr(pos), _ptr(freqs)),
                        (Qo, Q, pos, freqs, Ko, K))


def rope(Qo, Q, pos, freqs, Ko=None, K=None, sections=None, layout="halves", inverse=False,
         stream=None):
    """Rotate queries (and keys) by their positions: Q/Qo [B][Hq][S][D], K/Ko [B][Hkv][S][D] (fp16,
    bf16 or fp32; a result may be its input). Pair i of a head turns by pos·freqs[i]: ``freqs``
    float64 on the GPU, one per pair, its length the number of pairs (the rest of the head is
    copied); ``pos`` int32 [B or 1][S], or [axes][B or 1][S] with ``sections`` the pairs of each
    axis. ``layout``: pair i is elements i and i + pairs ("halves") or 2i and 2i + 1 ("pairs").
    ``inverse`` turns back, which is also the gradient: dQ = rope(dQo, inverse)."""
    prepare_rope(Qo, Q, pos, freqs, Ko, K, sections, layout, inverse)(stream)
    return Qo if Ko is None else (Qo, Ko)


def _paged_desc(op, Kc, Vc, block_table, seq_lens, cu_q, max_q, tokens, heads_q, prefix_len):
    torch = _torch()
    if Kc.dim() != 4 or Kc.shape != Vc.shape:
        _refuse(op, f"the caches are [pages][page_size][Hkv][D] of one shape, got {tuple(Kc.shape)} "
                    f"and {tuple(Vc.shape)}")
    if Kc.dtype != Vc.dtype:
        _refuse(op, "the caches must share a dtype", LVB_ERR_UNSUPPORTED)
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or (
            block_table.shape[1] > 1 and block_table.stride(1) != 1):
        _refuse(op, "block_table is int32 [B][pages per sequence], its rows contiguous")
    B = block_table.shape[0]
    if B > 1 and block_table.stride(0) < block_table.shape[1]:    # (0 is "packed" in the descriptor)
        _refuse(op, "block_table: stride below its width (an expanded table needs a copy)")
    _list_of(op, "seq_lens", seq_lens, torch.int32)
    if seq_lens.shape[0] != B:
        _refuse(op, f"seq_lens has {seq_lens.shape[0]} entries, block_table {B} rows")
    if cu_q is not None:
        _list_of(op, "cu_q", cu_q, torch.int32)
        if cu_q.shape[0] != B + 1:
            _refuse(op, f"cu_q has {cu_q.shape[0]} entries, needs {B + 1}")
        if max_q is None:
            _refuse(op, "cu_q without max_q: the most query rows of a sequence, known on the host")
    else:
        if max_q is None:
            max_q = tokens // B if B else 0
        if B * max_q != tokens:
            _refuse(op, f"{tokens} rows for {B} sequences of {max_q}: pass cu_q")
    d = lvb_paged_desc()
    d.dtype = dtype_of(Kc)
    d.batch, d.heads_q, d.heads_kv, d.head_dim = B, heads_q, Kc.shape[2], Kc.shape[3]
    d.tokens, d.max_q = tokens, int(max_q)
    d.page_size, d.num_pages = Kc.shape[1], Kc.shape[0]
    d.table_width = block_table.shape[1]
    d.table_stride = block_table.stride(0) if B > 1 else block_table.shape[1]
    d.prefix_len = int(prefix_len)
    d.scale = float(Kc.shape[3]) ** -0.5
    d.kc_stride[:] = _rows(op, "Kc", Kc, Kc.shape[:3])
    d.vc_stride[:] = _rows(op, "Vc", Vc, Vc.shape[:3])
    return d


def prepare_kv_append(Kc, Vc, K, V, block_table, seq_lens, cu_q=None, max_q=None, Qo=None, Q=None,
                      pos=None, freqs=None, sections=None, layout="halves",
                      prefix_len=0) -> PreparedCall:
    """``kv_append`` described once (see ``PreparedCall``)."""
    op = "lvb_kv_append"
    torch = _torch()
    if (Q is None) != (Qo is None):
        _refuse(op, "Q and Qo come together")
    if K.dim() != 3:
        _refuse(op, f"K and V are [tokens][Hkv][D], got {tuple(K.shape)}")
    T = K.shape[0]
    heads_q = Q.shape[1] if Q is not None and Q.dim() == 3 else 0
    d = lvb_append_desc()
    d.paged = _paged_desc(op, Kc, Vc, block_table, seq_lens, cu_q, max_q, T, heads_q, prefix_len)
    Hkv, D = Kc.shape[2], Kc.shape[3]
    for field_, name, t in (("k_stride", "K", K), ("v_stride", "V", V)):
        if tuple(t.shape) != (T, Hkv, D) or t.dtype != Kc.dtype:
            _refuse(op, f"{name} must be [{T}][{Hkv}][{D}] of the cache's dtype")
        getattr(d, field_)[:] = _rows(op, name, t, (T, Hkv))
    if Q is not None:
        for field_, name, t in (("q_stride", "Q", Q), ("o_stride", "Qo", Qo)):
            if t.dim() != 3 or tuple(t.shape) != (T, heads_q, D) or t.dtype != Kc.dtype:
                _refuse(op, f"{name} must be [{T}][Hq][{D}] of the cache's dtype")
            getattr(d.paged, field_)[:] = _rows(op, name, t, (T, heads_q))
    if freqs is not None:
        d.rot = _rotation(op, freqs, sections, layout, False)
        if pos is not None:
            p = pos if pos.dim() == 2 else pos.unsqueeze(0)
            if (pos.dtype != torch.int32 or tuple(p.shape) != (d.rot.n_axes, T)
                    or (T > 1 and p.stride(1) != 1)):
                _refuse(op, f"pos is int32 [{T}], or [{d.rot.n_axes}][{T}] for several axes, "
                            "its rows contiguous")
            d.pos_stride = p.stride(0)
        elif d.rot.n_axes != 1:
            _refuse(op, "several axes need pos")
    elif pos is not None or Q is not None:
        _refuse(op, "pos or Q without freqs")
    check(lib.lvb_kv_append_check(C.byref(d)))
    keep = (Kc, Vc, K, V, Q, Qo, block_table, seq_lens, cu_q, pos, freqs)
    _on_current_device(op, dict(zip(("Kc", "Vc", "K", "V", "Q", "Qo", "block_table", "seq_lens",
                                     "cu_q", "pos", "freqs"), keep)))
    return PreparedCall(lib.lvb_kv_append, d, tuple(_ptr(t) for t in keep), keep)


def kv_append(Kc, Vc, K, V, block_table, seq_lens, cu_q=None, max_q=None, Qo=None, Q=None, pos=None,
              freqs=None, sections=None, layout="halves", prefix_len=0, stream=None):
    """Write the new tokens' keys and values into a paged cache. Kc/Vc [pages][page_size][Hkv][D]
    (any strides), K/V [tokens][Hkv][D] packed by sequence: sequence b has rows cu_q[b] ..
    cu_q[b+1]-1 (at most ``max_q``; without ``cu_q`` all have the same number) and they become its
    last places, up to seq_lens[b] - 1 (``seq_lens`` counts them), place p in slot p % page_size of
    page block_table[b][p // page_size]. With ``freqs`` the keys are rotated on the way (as
    ``rope``; ``pos`` int32 [tokens] or [axes][tokens], by default prefix_len + place), and
    ``Q`` [tokens][Hq][D] beside them into ``Qo`` (which may be Q). A row whose place is negative (an
    idle entry of a padded batch) is left out. Lists are int32 on the GPU and read there: what they
    get wrong is reported by ``device_status`` (see include/lvb.h)."""
    prepare_kv_append(Kc, Vc, K, V, block_table, seq_lens, cu_q, max_q, Qo, Q, pos, freqs, sections,
                      layout, prefix_len)(stream)
    return Kc, Vc


def prepare_attention_paged(O, Q, Kc, Vc, block_table, seq_lens, cu_q=None, max_q=None, causal=True,
                            scale=None, lse=None, prefix_table=None, prefix_len=0) -> PreparedCall:
    """``attention_paged`` described once (see ``PreparedCall``)."""
    op = "lvb_attention_paged"
    torch = _torch()
    if Q.dim() != 3 or O.shape != Q.shape or Q.shape[2] != Kc.shape[-1]:
        _refuse(op, f"Q and O are [tokens][Hq][D], got {tuple(Q.shape)} and {tuple(O.shape)}")
    T, Hq, _ = Q.shape
    d = _paged_desc(op, Kc, Vc, block_table, seq_lens, cu_q, max_q, T, Hq, prefix_len)
    if not Q.dtype == O.dtype == Kc.dtype:
        _refuse(op, "Q, O and the caches must share a dtype", LVB_ERR_UNSUPPORTED)
    d.causal = int(bool(causal))
    if scale is not None:
        d.scale = float(scale)
    d.q_stride[:] = _rows(op, "Q", Q, (T, Hq))
    d.o_stride[:] = _rows(op, "O", O, (T, Hq))
    if d.prefix_len > 0:
        if prefix_table is None:
            _refuse(op, "prefix_len without prefix_table")
        _list_of(op, "prefix_table", prefix_table, torch.int32,
                 -(-d.prefix_len // max(1, d.page_size)))
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (T, Hq)
                            or not lse.is_contiguous()):
        _refuse(op, f"lse must be contiguous float32 [{T}][{Hq}]")
    check(lib.lvb_attention_paged_check(C.byref(d)))
    keep = (Q, Kc, Vc, block_table, seq_lens, cu_q, prefix_table, O, lse)
    _on_current_device(op, dict(zip(("Q", "Kc", "Vc", "block_table", "seq_lens", "cu_q",
                                     "prefix_table", "O", "lse"), keep)))
    return PreparedCall(lib.lvb_attention_paged, d, tuple(_ptr(t) for t in keep), keep)


def attention_paged(O, Q, Kc, Vc, block_table, seq_lens, cu_q=None, max_q=None, causal=True,
                    scale=None, lse=None, prefix_table=None, prefix_len=0, stream=None):
    """Attention of packed queries over a paged cache: Q/O [tokens][Hq][D], the caches, the table and
    the lists as in ``kv_append`` (seq_lens counts the queries' own tokens). A query at place p
    sees places 0..p (``causal``; else all of its sequence's), and before them the ``prefix_len``
    keys whose pages ``prefix_table`` (int32) lists, which all sequences share (read once for
    all of them, or in front of each one's own where that takes less time). Optional ``lse``
    float32 [tokens][Hq]. Rows that see no key give O = 0 and lse = -inf; rows behind cu_q[B] are
    left as they were."""
    prepare_attention_paged(O, Q, Kc, Vc, block_table, seq_lens, cu_q, max_q, causal, scale, lse,
                            prefix_table, prefix_len)(stream)
    return O


def attention_paged_plan(B, Hq, Hkv, tokens, max_q, page_size, table_width, D=128, dtype=BF16,
                         causal=True, prefix_len=0, sm_count=148) -> lvb_paged_plan:
    """How lvb_attention_paged runs a call of these extents (host only, no GPU)."""
    d = lvb_paged_desc()
    d.dtype, d.causal = dtype, int(bool(causal))
    d.batch, d.heads_q, d.heads_kv, d.head_dim = B, Hq, Hkv, D
    d.tokens, d.max_q, d.page_size, d.num_pages = tokens, max_q, page_size, 1
    d.table_width, d.prefix_len, d.scale = table_width, prefix_len, float(D) ** -0.5
    p = lvb_paged_plan()
    check(lib.lvb_attention_paged_plan_for(C.byref(d), sm_count, C.byref(p)))
    return p


def attention_available() -> bool:
    return True


def device_status(stream=None):
    """Synchronise and read/clear the device status word: (code, where, block)."""
    code, where, block = C.c_int32(), C.c_int32(), C.c_int32()
    check(lib.lvb_device_status(_stream_ptr(stream), C.byref(code), C.byref(where), C.byref(block)))
    return code.value, where.value, block.value


def gemm_noalloc_status(stream=None):
    """Synchronise and read/clear lvb_gemm_noalloc's own status word: (code, where, block)."""
    code, where, block = C.c_int32(), C.c_int32(), C.c_int32()
    check(lib.lvb_gemm_noalloc_status(_stream_ptr(stream), C.byref(code), C.byref(where),
                                      C.byref(block)))
    return code.value, where.value, block.value


def selftest_wait_timeout(ms: int = 50, stream=None) -> None:
    """Enqueue the failure-path self-test (a wait nothing satisfies, limited to ``ms``)."""
    check(lib.lvb_selftest_wait_timeout(int(ms), _stream_ptr(stream)))


def set_wait_timeout_ms(ms: int) -> None:
    check(lib.lvb_set_wait_timeout_ms(int(ms)))


def abi_version() -> int:
    return lib.lvb_abi_version()
