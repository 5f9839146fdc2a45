"""ctypes binding of ``libiqk_b200.so`` plus the reference's geometry guards.

The CUDA library is the product: this module loads it (failing loudly when it
is missing -- there is no CPU or eager fallback), declares the C ABI of
``include/iqk_b200.h``, and maps status codes onto the reference's exception
classes. The guard functions keep the reference's names and messages
(``src/mlx_iqk/kernels.py:100-128``).
"""

from __future__ import annotations

import ctypes
import functools
import os
from pathlib import Path

import torch
from torch.autograd import forward_ad

from .format import (DENSE_MEMBER_IDS, MEMBER_IDS, IqkFormatError, check_dense_member,
                     check_member, check_row_width)

ROWS_PER_TG = 16
"""Output rows one decode work unit (a warp) covers; out_features must tile it."""

SUPPORTED_IN_FEATURES = (2048, 4096)
"""Input widths the kernels are sized for: the down and gate/up widths."""

IQ2_MEMBERS = ("iq2_ks", "iq2_k")
"""Members the reference records sorted/union GEMV formulations for."""

LIB_PATH = Path(__file__).resolve().parent / "libiqk_b200.so"

IQK_OK = 0
_STATUS_NAMES = {
    1: "IQK_ERR_MEMBER", 2: "IQK_ERR_WIDTH", 3: "IQK_ERR_GEOMETRY", 4: "IQK_ERR_ARGUMENT",
    5: "IQK_ERR_ALIGNMENT", 6: "IQK_ERR_WORKSPACE", 7: "IQK_ERR_CUDA", 8: "IQK_ERR_DEVICE",
}
DEVERR_EXPERT, DEVERR_TOKEN, DEVERR_NONFINITE, DEVERR_TIMEOUT = 1, 2, 4, 8
DTYPE_IDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class IqkKernelError(RuntimeError):
    """Geometry the kernels are not sized for (reference class name)."""


class IqkRuntimeError(RuntimeError):
    """Operand/stream contract violation or a failed launch (reference class name)."""


def check_gemv_geometry(in_features: int, out_features: int) -> tuple[int, int]:
    """Reject any geometry the decode GEMV does not cover, before launching."""
    n = check_row_width(in_features)
    if n not in SUPPORTED_IN_FEATURES:
        raise IqkKernelError(
            f"the decode gemv is sized per input width and covers "
            f"{SUPPORTED_IN_FEATURES}, got {in_features}")
    out = int(out_features)
    if out <= 0 or out % ROWS_PER_TG:
        raise IqkKernelError(
            f"out_features {out_features} is not a positive multiple of {ROWS_PER_TG}")
    return n, out


def check_dequant_geometry(in_features: int, out_features: int) -> tuple[int, int]:
    """Reject any geometry the stacked dequantization does not cover."""
    n = check_row_width(in_features)
    if n not in SUPPORTED_IN_FEATURES:
        raise IqkKernelError(
            f"the dequantization is sized per input width and covers "
            f"{SUPPORTED_IN_FEATURES}, got {in_features}")
    out = int(out_features)
    if out <= 0:
        raise IqkKernelError(f"out_features {out_features} is not positive")
    return n, out


# ------------------------------------------------------------------ loading

_LIB = None


def library() -> ctypes.CDLL:
    """The loaded CUDA library; raises if it was never built."""
    global _LIB
    if _LIB is not None:
        return _LIB
    path = Path(os.environ.get("IQK_B200_LIB", LIB_PATH))
    if not path.exists():
        raise IqkRuntimeError(
            f"{path} is not built; run `python -c 'import __graft_entry__ as g; g.build()'` "
            "(the IQ_K kernels have no CPU fallback)")
    lib = ctypes.CDLL(str(path))
    vp, i64, i32, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
    lib.iqk_status_string.argtypes = [i32]
    lib.iqk_status_string.restype = ctypes.c_char_p
    lib.iqk_abi_version.restype = i32
    lib.iqk_check_device.restype = i32
    lib.iqk_check_bounded_wait.argtypes = [i64, vp, vp]
    lib.iqk_check_bounded_wait.restype = i32
    lib.iqk_dequant.argtypes = [i32, vp, i64, i64, i64, i64, i64, i32, vp, vp]
    lib.iqk_dequant.restype = i32
    lib.iqk_dense_dequant.argtypes = [i32, vp, i64, i64, i64, i64, i32, vp, vp]
    lib.iqk_dense_dequant.restype = i32
    lib.iqk_dense_gemv.argtypes = [i32, vp, i64, vp, i64, i64, vp, i32, vp]
    lib.iqk_dense_gemv.restype = i32
    lib.iqk_pack.argtypes = [i32, vp, i64, i64, vp, vp]
    lib.iqk_pack.restype = i32
    lib.iqk_gemv_workspace_bytes.argtypes = [i32, i64, i64, i64]
    lib.iqk_gemv_workspace_bytes.restype = sz
    lib.iqk_gemv_workspace_min_bytes.argtypes = [i32, i64, i64, i64]
    lib.iqk_gemv_workspace_min_bytes.restype = sz
    lib.iqk_gemv.argtypes = [i32, vp, i32, i64, vp, i64, i64, i64, vp, vp, i64, vp, i32, vp,
                             sz, vp]
    lib.iqk_gemv.restype = i32
    lib.iqk_gemv_prepare.argtypes = [vp, i32, i64, i64, i64, vp, vp, i64, vp, sz, vp]
    lib.iqk_gemv_prepare.restype = i32
    lib.iqk_gemv_run.argtypes = [i32, vp, i64, i64, i64, i64, i64, vp, i32, vp, sz, vp]
    lib.iqk_gemv_run.restype = i32
    lib.iqk_gemv_floor_run.argtypes = [i32, vp, i64, i64, i64, i64, i64, vp, i32, vp, sz, vp]
    lib.iqk_gemv_floor_run.restype = i32
    lib.iqk_gemv_glu_run.argtypes = [i32, vp, vp, i64, i64, i64, i64, i64, vp, vp, vp, sz, vp]
    lib.iqk_gemv_glu_run.restype = i32
    lib.iqk_swiglu_rows.argtypes = [vp, vp, vp, i64, i64, vp, vp]
    lib.iqk_swiglu_rows.restype = i32
    lib.iqk_dequant_floor.argtypes = [i32, vp, i64, i64, i64, i64, i64, i32, vp, vp]
    lib.iqk_dequant_floor.restype = i32
    lib.iqk_read_error.argtypes = [vp, i64, i64, i64, ctypes.POINTER(ctypes.c_int32), vp]
    lib.iqk_read_error.restype = i32
    lib.iqk_grouped_workspace_bytes.argtypes = [i64, i64, i64]
    lib.iqk_grouped_workspace_bytes.restype = sz
    lib.iqk_grouped_gemm.argtypes = [i32, vp, i32, i64, vp, i64, i64, i64, vp, vp, i64, vp, i32,
                                     vp, sz, vp]
    lib.iqk_grouped_gemm.restype = i32
    lib.iqk_grouped_prepare.argtypes = [vp, i32, i64, i64, i64, vp, vp, i64, vp, sz, vp]
    lib.iqk_grouped_prepare.restype = i32
    lib.iqk_grouped_run.argtypes = [i32, vp, i64, i64, i64, i64, vp, i32, vp, sz, vp]
    lib.iqk_grouped_run.restype = i32
    lib.iqk_grouped_run_range.argtypes = [i32, vp, i64, i64, i64, i64, i64, i64, vp, i32, vp,
                                          sz, vp]
    lib.iqk_grouped_run_range.restype = i32
    lib.iqk_grouped_read_error.argtypes = [vp, ctypes.POINTER(ctypes.c_int32), vp]
    lib.iqk_grouped_read_error.restype = i32
    lib.iqk_gemv_static_max_bytes.restype = sz
    lib.iqk_gemv_static.argtypes = [i32, vp, i32, i64, vp, i64, i64, i64, vp, vp, i64, vp, i32,
                                    vp]
    lib.iqk_gemv_static.restype = i32
    lib.iqk_gemv_static_read_error.argtypes = [i64, i64, i64, ctypes.POINTER(ctypes.c_int32), vp]
    lib.iqk_gemv_static_read_error.restype = i32
    lib.iqk_grouped_prepare_shard.argtypes = [vp, i32, i64, i64, i64, vp, vp, i64, vp, sz, vp]
    lib.iqk_grouped_prepare_shard.restype = i32
    lib.iqk_pairs_swiglu.argtypes = [vp, vp, vp, i64, i64, i64, i64, vp, sz, vp, vp]
    lib.iqk_pairs_swiglu.restype = i32
    lib.iqk_pairs_combine.argtypes = [vp, vp, i64, i32, i64, i64, vp, i32, vp]
    lib.iqk_pairs_combine.restype = i32
    f32 = ctypes.c_float
    lib.iqk_narrow_indices.argtypes = [vp, i64, vp, vp]
    lib.iqk_narrow_indices.restype = i32
    lib.iqk_route.argtypes = [vp, i32, i64, i64, i64, vp, i32, i32, i32, f32, vp, vp, vp]
    lib.iqk_route.restype = i32
    lib.iqk_balance_workspace_bytes.argtypes = [i64, i64, i64]
    lib.iqk_balance_workspace_bytes.restype = sz
    lib.iqk_route_balanced.argtypes = [vp, i32, i64, i64, i64, vp, vp, i64, i32, i32, i32, f32,
                                       vp, vp, vp, vp, vp, vp, sz, vp]
    lib.iqk_route_balanced.restype = i32
    lib.iqk_route_backward.argtypes = [vp, i32, i64, i64, i64, vp, vp, i64, i32, i32, i32, f32,
                                       vp, vp, vp, vp, vp, vp]
    lib.iqk_route_backward.restype = i32
    lib.iqk_mx_quantize.argtypes = [vp, i32, i64, i64, i64, vp, vp, i64, vp]
    lib.iqk_mx_quantize.restype = i32
    lib.iqk_mx_dequantize.argtypes = [vp, vp, i64, i64, i64, vp, i32, vp]
    lib.iqk_mx_dequantize.restype = i32
    lib.iqk_mx_workspace_bytes.argtypes = [i64, i64, i64, i64]
    lib.iqk_mx_workspace_bytes.restype = sz
    lib.iqk_mx_linear.argtypes = [vp, i32, i64, i64, vp, vp, i64, i64, i64, vp, i32, vp, sz, vp]
    lib.iqk_mx_linear.restype = i32
    lib.iqk_mx_routed.argtypes = [vp, i32, i64, i64, vp, i64, vp, vp, i64, i64, i64, i64, vp, i32,
                                  vp, sz, vp]
    lib.iqk_mx_routed.restype = i32
    lib.iqk_mx_few_state_bytes.argtypes = []
    lib.iqk_mx_few_state_bytes.restype = sz
    lib.iqk_mx_few_state_bytes_for.argtypes = [i64]
    lib.iqk_mx_few_state_bytes_for.restype = sz
    lib.iqk_mx_few_fits.argtypes = [i64, i64, i64, i64, i32]
    lib.iqk_mx_few_fits.restype = i32
    lib.iqk_mx_few.argtypes = lib.iqk_mx_routed.argtypes
    lib.iqk_mx_few.restype = i32
    lib.iqk_mx_read_error.argtypes = [vp, ctypes.POINTER(ctypes.c_int32), vp]
    lib.iqk_mx_read_error.restype = i32
    lib.iqk_mx_take_errors.argtypes = [ctypes.POINTER(ctypes.c_int32), vp]
    lib.iqk_mx_take_errors.restype = i32
    lib.iqk_mx_error_word.argtypes = [ctypes.POINTER(vp)]
    lib.iqk_mx_error_word.restype = i32
    _LIB = lib
    return lib


def exported_symbols() -> list[str]:
    """C ABI entry points declared in include/iqk_b200.h."""
    return ["iqk_status_string", "iqk_abi_version", "iqk_check_device", "iqk_dequant",
            "iqk_gemv_workspace_bytes", "iqk_gemv_workspace_min_bytes", "iqk_gemv",
            "iqk_gemv_prepare", "iqk_gemv_run",
            "iqk_read_error", "iqk_grouped_workspace_bytes", "iqk_grouped_gemm",
            "iqk_grouped_prepare", "iqk_grouped_run", "iqk_grouped_read_error",
            "iqk_gemv_static_max_bytes", "iqk_gemv_static", "iqk_gemv_static_read_error",
            "iqk_grouped_prepare_shard",
            "iqk_pairs_swiglu", "iqk_pairs_combine", "iqk_gemv_floor_run",
            "iqk_dequant_floor", "iqk_grouped_run_range", "iqk_pack",
            "iqk_gemv_glu_run", "iqk_swiglu_rows", "iqk_check_bounded_wait",
            "iqk_dense_dequant", "iqk_dense_gemv",
            "iqk_narrow_indices", "iqk_route", "iqk_balance_workspace_bytes", "iqk_route_balanced",
            "iqk_route_backward", "iqk_mx_quantize", "iqk_mx_dequantize",
            "iqk_mx_workspace_bytes", "iqk_mx_linear", "iqk_mx_routed", "iqk_mx_read_error",
            "iqk_mx_take_errors", "iqk_mx_error_word",
            "iqk_mx_few_state_bytes", "iqk_mx_few_state_bytes_for", "iqk_mx_few_fits", "iqk_mx_few"]


def check_bounded_wait(limit_ns: int, device: torch.device) -> int:
    """``iqk_check_bounded_wait``: the device error bits a wait that nothing
    satisfies leaves after ``limit_ns`` (IQK_DEVERR_TIMEOUT expected)."""
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    raise_for_status(library().iqk_check_bounded_wait(limit_ns, flags.data_ptr(),
                                                      stream_handle(device)),
                     "iqk_check_bounded_wait")
    return int(flags.item())


def raise_for_status(status: int, what: str) -> None:
    if status == IQK_OK:
        return
    msg = f"{what}: {library().iqk_status_string(status).decode()} ({_STATUS_NAMES.get(status, status)})"
    if status == 1:
        raise IqkFormatError(msg)
    if status in (2, 3):
        raise IqkKernelError(msg)
    raise IqkRuntimeError(msg)


_DEVICE_OK: dict[int, bool] = {}


def check_device(device: torch.device) -> None:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _DEVICE_OK:
        with torch.cuda.device(idx):
            raise_for_status(library().iqk_check_device(), "device check")
        _DEVICE_OK[idx] = True


def check_current(device: torch.device) -> None:
    """The kernels launch on the current device: refuse tensors of another one."""
    if device.index != torch.cuda.current_device():
        raise IqkRuntimeError(
            f"tensors on {device}, but the current device is {torch.cuda.current_device()}")
    check_device(device)


def refuse_tangent(t: torch.Tensor, what: str) -> None:
    """The kernels have no forward-mode derivative: a dual tensor's tangent would
    be lost without a word, since a call by address does not see it. Outside a
    dual level, the common case, this is one comparison (unpack_dual takes 0.4 us)."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise IqkRuntimeError(f"{what} carries a tangent: there is no forward-mode derivative")


def stream_handle(device: torch.device) -> int:
    """The device's current stream as a handle; the raw query makes no Stream
    object (0.1 us for 2.2 us a call)."""
    index = device.index
    return torch._C._cuda_getCurrentRawStream(
        torch.cuda.current_device() if index is None else index)


_PTR_ARRAYS: dict[tuple, ctypes.Array] = {}


def ptr_array(tensors) -> ctypes.Array:
    """The streams' device pointers as a C array (cached per pointer tuple:
    a module's streams keep their storage between calls)."""
    key = tuple(t.data_ptr() for t in tensors)
    arr = _PTR_ARRAYS.get(key)
    if arr is None:
        if len(_PTR_ARRAYS) > 256:
            _PTR_ARRAYS.clear()
        arr = (ctypes.c_void_p * len(key))(*key)
        _PTR_ARRAYS[key] = arr
    return arr


def pack(member: str, wire: torch.Tensor, in_features: int, streams) -> None:
    """``iqk_pack``: ik wire rows [rows, ggml row bytes] (uint8, on the device)
    into ``streams`` (component order, each [rows, length] viewed flat)."""
    check_device(wire.device)
    status = library().iqk_pack(MEMBER_IDS[check_member(member)], wire.data_ptr(),
                                wire.shape[0], in_features, ptr_array(streams),
                                stream_handle(wire.device))
    raise_for_status(status, "iqk_pack")


def dequant(member: str, streams, num_experts: int, out_features: int, in_features: int,
            row_start: int, rows: int, out: torch.Tensor) -> torch.Tensor:
    """``iqk_dequant`` into ``out`` [E, rows, in] on the current stream."""
    lib = library()
    check_device(out.device)
    status = lib.iqk_dequant(MEMBER_IDS[check_member(member)], ptr_array(streams), num_experts,
                             out_features, in_features, row_start, rows,
                             DTYPE_IDS[out.dtype], out.data_ptr(), stream_handle(out.device))
    raise_for_status(status, "iqk_dequant")
    return out


def dense_dequant(member: str, streams, out_features: int, in_features: int, row_start: int,
                  rows: int, out: torch.Tensor) -> torch.Tensor:
    """``iqk_dense_dequant``: rows [row_start, row_start + rows) of a dense
    matrix into ``out`` [rows, in] (f32, f16 or bf16)."""
    check_device(out.device)
    status = library().iqk_dense_dequant(DENSE_MEMBER_IDS[check_dense_member(member)],
                                         ptr_array(streams), out_features, in_features,
                                         row_start, rows, DTYPE_IDS[out.dtype], out.data_ptr(),
                                         stream_handle(out.device))
    raise_for_status(status, "iqk_dense_dequant")
    return out


def dense_gemv(member: str, x: torch.Tensor, streams, out_features: int, in_features: int,
               y: torch.Tensor) -> torch.Tensor:
    """``iqk_dense_gemv``: ``y [T, out] = x [T, in] W^T`` for f16 ``x``; ``y``
    f16 or f32."""
    check_device(y.device)
    if x.dtype != torch.float16 or not x.is_contiguous():
        raise IqkRuntimeError("the dense gemv takes contiguous fp16 activations")
    status = library().iqk_dense_gemv(DENSE_MEMBER_IDS[check_dense_member(member)],
                                      x.data_ptr(), x.shape[0], ptr_array(streams),
                                      out_features, in_features, y.data_ptr(),
                                      DTYPE_IDS[y.dtype], stream_handle(y.device))
    raise_for_status(status, "iqk_dense_gemv")
    return y


@functools.lru_cache(maxsize=1024)
def gemv_workspace_bytes(member: str, in_features: int, x_rows: int, pairs: int) -> int:
    return int(library().iqk_gemv_workspace_bytes(MEMBER_IDS[member], in_features, x_rows, pairs))


def gemv_workspace_min_bytes(member: str, in_features: int, x_rows: int, pairs: int) -> int:
    """The smallest workspace the GEMV accepts (no split slots: whole items)."""
    return int(library().iqk_gemv_workspace_min_bytes(MEMBER_IDS[member], in_features, x_rows,
                                                      pairs))


def gemv(member: str, x: torch.Tensor, streams, num_experts: int, out_features: int,
         in_features: int, sel: torch.Tensor, tok: torch.Tensor | None, y: torch.Tensor,
         workspace: torch.Tensor | None = None, stream: int | None = None) -> torch.Tensor:
    """``iqk_gemv``: x [x_rows, in], sel/tok int32 [pairs], y [pairs, out]; on
    ``stream`` (a CUDA stream handle), else the device's current stream."""
    lib = library()
    check_device(y.device)
    pairs = sel.numel()
    x_rows = x.shape[0]
    need = gemv_workspace_bytes(member, in_features, x_rows, pairs)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=y.device)
    status = lib.iqk_gemv(
        MEMBER_IDS[member], x.data_ptr(), DTYPE_IDS[x.dtype], x_rows, ptr_array(streams),
        num_experts, out_features, in_features, sel.data_ptr(),
        None if tok is None else tok.data_ptr(), pairs, y.data_ptr(), DTYPE_IDS[y.dtype],
        workspace.data_ptr(), workspace.numel(),
        stream_handle(y.device) if stream is None else stream)
    raise_for_status(status, "iqk_gemv")
    return y


def gemv_prepare(x: torch.Tensor, num_experts: int, in_features: int, sel: torch.Tensor,
                 tok: torch.Tensor | None, workspace: torch.Tensor) -> torch.Tensor:
    """``iqk_gemv_prepare``: activation digit planes + routing into ``workspace``."""
    lib = library()
    check_device(workspace.device)
    status = lib.iqk_gemv_prepare(
        x.data_ptr(), DTYPE_IDS[x.dtype], x.shape[0], in_features, num_experts,
        sel.data_ptr(), None if tok is None else tok.data_ptr(), sel.numel(),
        workspace.data_ptr(), workspace.numel(), stream_handle(workspace.device))
    raise_for_status(status, "iqk_gemv_prepare")
    return workspace


def gemv_run(member: str, streams, num_experts: int, out_features: int, in_features: int,
             x_rows: int, pairs: int, y: torch.Tensor, workspace: torch.Tensor) -> torch.Tensor:
    """``iqk_gemv_run``: one projection over a prepared workspace into ``y``."""
    lib = library()
    status = lib.iqk_gemv_run(
        MEMBER_IDS[member], ptr_array(streams), num_experts, out_features, in_features, x_rows,
        pairs, y.data_ptr(), DTYPE_IDS[y.dtype], workspace.data_ptr(), workspace.numel(),
        stream_handle(y.device))
    raise_for_status(status, "iqk_gemv_run")
    return y


def gemv_glu_run(member: str, gate_streams, up_streams, num_experts: int, out_features: int,
                 in_features: int, x_rows: int, pairs: int, weight: torch.Tensor | None,
                 h: torch.Tensor, workspace: torch.Tensor) -> torch.Tensor:
    """``iqk_gemv_glu_run``: h [pairs, out] float32 = silu(gate) * up * weight."""
    status = library().iqk_gemv_glu_run(
        MEMBER_IDS[member], ptr_array(gate_streams), ptr_array(up_streams), num_experts,
        out_features, in_features, x_rows, pairs,
        None if weight is None else weight.data_ptr(), h.data_ptr(), workspace.data_ptr(),
        workspace.numel(), stream_handle(h.device))
    raise_for_status(status, "iqk_gemv_glu_run")
    return h


def swiglu_rows(g: torch.Tensor, u: torch.Tensor, weight: torch.Tensor | None,
                h: torch.Tensor) -> torch.Tensor:
    """``iqk_swiglu_rows``: h = silu(g) * u * weight[row], float32 [rows, cols]."""
    status = library().iqk_swiglu_rows(
        g.data_ptr(), u.data_ptr(), None if weight is None else weight.data_ptr(), g.shape[0],
        g.shape[1], h.data_ptr(), stream_handle(h.device))
    raise_for_status(status, "iqk_swiglu_rows")
    return h


def gemv_floor_run(member: str, streams, num_experts: int, out_features: int,
                   in_features: int, x_rows: int, pairs: int, y: torch.Tensor,
                   workspace: torch.Tensor) -> torch.Tensor:
    """``iqk_gemv_floor_run``: the GEMV's address floor (benchmark only)."""
    status = library().iqk_gemv_floor_run(
        MEMBER_IDS[member], ptr_array(streams), num_experts, out_features, in_features, x_rows,
        pairs, y.data_ptr(), DTYPE_IDS[y.dtype], workspace.data_ptr(), workspace.numel(),
        stream_handle(y.device))
    raise_for_status(status, "iqk_gemv_floor_run")
    return y


def dequant_floor(member: str, streams, num_experts: int, out_features: int, in_features: int,
                  row_start: int, rows: int, out: torch.Tensor) -> torch.Tensor:
    """``iqk_dequant_floor``: the dequantization's address floor (benchmark only)."""
    status = library().iqk_dequant_floor(MEMBER_IDS[check_member(member)], ptr_array(streams),
                                         num_experts, out_features, in_features, row_start,
                                         rows, DTYPE_IDS[out.dtype], out.data_ptr(),
                                         stream_handle(out.device))
    raise_for_status(status, "iqk_dequant_floor")
    return out


def gemv_static(member: str, x: torch.Tensor, streams, num_experts: int, out_features: int,
                in_features: int, sel: torch.Tensor, tok: torch.Tensor | None,
                y: torch.Tensor) -> torch.Tensor:
    """``iqk_gemv_static``: as :func:`gemv`, scratch in the library's static device array."""
    lib = library()
    check_device(y.device)
    status = lib.iqk_gemv_static(
        MEMBER_IDS[member], x.data_ptr(), DTYPE_IDS[x.dtype], x.shape[0], ptr_array(streams),
        num_experts, out_features, in_features, sel.data_ptr(),
        None if tok is None else tok.data_ptr(), sel.numel(), y.data_ptr(), DTYPE_IDS[y.dtype],
        stream_handle(y.device))
    raise_for_status(status, "iqk_gemv_static")
    return y


def gemv_static_read_error(in_features: int, x_rows: int, pairs: int,
                           device: torch.device | None = None) -> int:
    """``iqk_gemv_static_read_error``: the device error bits of the last
    ``iqk_gemv_static`` call of this geometry on the current device."""
    flags = ctypes.c_int32(0)
    dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    raise_for_status(library().iqk_gemv_static_read_error(in_features, x_rows, pairs,
                                                          ctypes.byref(flags),
                                                          stream_handle(dev)),
                     "iqk_gemv_static_read_error")
    return int(flags.value)


GROUPED_MEMBERS = ("iq2_ks", "iq2_k", "iq1_s_r4")
"""Members the tensor-core grouped GEMM (prefill route) covers."""


def grouped_workspace_bytes(in_features: int, num_experts: int, pairs: int) -> int:
    return int(library().iqk_grouped_workspace_bytes(in_features, num_experts, pairs))


def grouped(member: str, x: torch.Tensor, streams, num_experts: int, out_features: int,
            in_features: int, sel: torch.Tensor, tok: torch.Tensor | None, y: torch.Tensor,
            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``iqk_grouped_gemm``: x [x_rows, in], sel/tok int32 [pairs], y [pairs, out]."""
    lib = library()
    check_device(y.device)
    pairs = sel.numel()
    need = grouped_workspace_bytes(in_features, num_experts, pairs)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=y.device)
    status = lib.iqk_grouped_gemm(
        MEMBER_IDS[member], x.data_ptr(), DTYPE_IDS[x.dtype], x.shape[0], ptr_array(streams),
        num_experts, out_features, in_features, sel.data_ptr(),
        None if tok is None else tok.data_ptr(), pairs, y.data_ptr(), DTYPE_IDS[y.dtype],
        workspace.data_ptr(), workspace.numel(), stream_handle(y.device))
    raise_for_status(status, "iqk_grouped_gemm")
    return y


def grouped_prepare(x: torch.Tensor, num_experts: int, in_features: int, sel: torch.Tensor,
                    tok: torch.Tensor | None, workspace: torch.Tensor,
                    shard: bool = False) -> torch.Tensor:
    """``iqk_grouped_prepare``; with ``shard`` ``iqk_grouped_prepare_shard``
    (pairs whose expert lies outside [0, num_experts) are another rank's:
    skipped, no error, their output rows left untouched)."""
    lib = library()
    check_device(workspace.device)
    fn = lib.iqk_grouped_prepare_shard if shard else lib.iqk_grouped_prepare
    status = fn(
        x.data_ptr(), DTYPE_IDS[x.dtype], x.shape[0], in_features, num_experts,
        sel.data_ptr(), None if tok is None else tok.data_ptr(), sel.numel(),
        workspace.data_ptr(), workspace.numel(), stream_handle(workspace.device))
    raise_for_status(status, "iqk_grouped_prepare_shard" if shard else "iqk_grouped_prepare")
    return workspace


def grouped_run(member: str, streams, num_experts: int, out_features: int, in_features: int,
                pairs: int, y: torch.Tensor, workspace: torch.Tensor) -> torch.Tensor:
    lib = library()
    status = lib.iqk_grouped_run(
        MEMBER_IDS[member], ptr_array(streams), num_experts, out_features, in_features, pairs,
        y.data_ptr(), DTYPE_IDS[y.dtype], workspace.data_ptr(), workspace.numel(),
        stream_handle(y.device))
    raise_for_status(status, "iqk_grouped_run")
    return y


def grouped_run_range(member: str, streams, num_experts: int, out_features: int,
                      in_features: int, pairs: int, row_start: int, rows: int, y: torch.Tensor,
                      workspace: torch.Tensor) -> torch.Tensor:
    """``iqk_grouped_run_range``: output rows [row_start, row_start + rows) of
    every expert over a prepared workspace into ``y`` [pairs, rows]."""
    status = library().iqk_grouped_run_range(
        MEMBER_IDS[member], ptr_array(streams), num_experts, out_features, in_features, pairs,
        row_start, rows, y.data_ptr(), DTYPE_IDS[y.dtype], workspace.data_ptr(),
        workspace.numel(), stream_handle(y.device))
    raise_for_status(status, "iqk_grouped_run_range")
    return y


def pairs_swiglu(g: torch.Tensor, u: torch.Tensor, w: torch.Tensor, in_features: int,
                 num_experts: int, workspace: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
    """``iqk_pairs_swiglu``: h[q] = bf16((silu(g[q]) * u[q]) * w[q]) for the pairs
    routed by ``workspace`` (prepared with ``in_features`` and ``num_experts``)."""
    pairs, inter = g.shape
    status = library().iqk_pairs_swiglu(
        g.data_ptr(), u.data_ptr(), w.data_ptr(), inter, in_features, num_experts, pairs,
        workspace.data_ptr(), workspace.numel(), h.data_ptr(), stream_handle(h.device))
    raise_for_status(status, "iqk_pairs_swiglu")
    return h


def pairs_combine(y: torch.Tensor, sel: torch.Tensor, top_k: int, num_experts: int,
                  out: torch.Tensor) -> torch.Tensor:
    """``iqk_pairs_combine``: out[r] = sum_j y[r*k + j] over the slots of row r
    whose sel lies in [0, num_experts)."""
    rows, hidden = out.shape
    status = library().iqk_pairs_combine(
        y.data_ptr(), sel.data_ptr(), rows, top_k, num_experts, hidden, out.data_ptr(),
        DTYPE_IDS[out.dtype], stream_handle(out.device))
    raise_for_status(status, "iqk_pairs_combine")
    return out


def grouped_read_error(workspace: torch.Tensor) -> int:
    flags = ctypes.c_int32(0)
    raise_for_status(library().iqk_grouped_read_error(workspace.data_ptr(), ctypes.byref(flags),
                                                      stream_handle(workspace.device)),
                     "iqk_grouped_read_error")
    return int(flags.value)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def expert_indices(indices: torch.Tensor) -> torch.Tensor:
    """``indices`` as the contiguous int32 that the kernels read. What 32 bits do not
    hold stays outside the experts (``iqk_narrow_indices``) and does not wrap into them."""
    if indices.dtype == torch.int32:
        return indices.contiguous()
    if indices.dtype.itemsize < 4 or not indices.is_cuda:
        return indices.to(torch.int32).contiguous()
    wide = indices.to(torch.int64).contiguous()
    check_current(wide.device)
    out = wide.new_empty(wide.shape, dtype=torch.int32)
    status = library().iqk_narrow_indices(wide.data_ptr(), wide.numel(), out.data_ptr(),
                                          stream_handle(wide.device))
    if status:
        raise_for_status(status, "iqk_narrow_indices")
    return out


@functools.lru_cache(maxsize=1024)
def balance_workspace_bytes(tokens: int, experts: int, segments: int) -> int:
    return int(library().iqk_balance_workspace_bytes(tokens, experts, segments))


def route(rows: torch.Tensor, mask, top_k: int, scoring: int, renormalize: bool, scale: float):
    """``iqk_route`` over logits ``rows [tokens, experts]``: ``(indices, weights)``."""
    dev = rows.device
    tokens, experts = rows.shape
    indices = rows.new_empty((tokens, top_k), dtype=torch.int32)
    weights = rows.new_empty((tokens, top_k), dtype=torch.float32)
    status = library().iqk_route(
        rows.data_ptr(), DTYPE_IDS[rows.dtype], tokens, experts, rows.stride(0), _ptr(mask),
        top_k, scoring, renormalize, scale, indices.data_ptr(), weights.data_ptr(),
        stream_handle(dev))
    if status:
        raise_for_status(status, "iqk_route")
    return indices, weights


def route_balanced(rows: torch.Tensor, mask, offsets, top_k: int, scoring: int,
                   renormalize: bool, scale: float, indices=None, keep_slope: bool = False):
    """``iqk_route_balanced``: ``(indices, weights, loss, counts, slope)``. With
    ``indices`` given (a choice already made) weights are None. ``slope``
    [segments, experts], which the backward call reads, is a tensor of its own when it
    is to be kept, so that the workspace is not; else None, and lies in the workspace."""
    dev = rows.device
    tokens, experts = rows.shape
    segments = 1 if offsets is None else offsets.numel() - 1
    weights = None
    if indices is None:
        indices = rows.new_empty((tokens, top_k), dtype=torch.int32)
        weights = rows.new_empty((tokens, top_k), dtype=torch.float32)
    need = balance_workspace_bytes(tokens, experts, segments)
    slope, extra = None, 4 * segments * experts
    if keep_slope:
        slope, extra = rows.new_empty((segments, experts), dtype=torch.float32), 0
    ws = rows.new_empty(need + extra, dtype=torch.uint8)
    loss = rows.new_empty((), dtype=torch.float32)
    counts = rows.new_empty((segments, experts), dtype=torch.int32)
    base = ws.data_ptr()
    status = library().iqk_route_balanced(
        rows.data_ptr(), DTYPE_IDS[rows.dtype], tokens, experts, rows.stride(0), _ptr(mask),
        _ptr(offsets), segments, top_k, scoring, renormalize, scale, indices.data_ptr(),
        _ptr(weights), loss.data_ptr(), counts.data_ptr(),
        slope.data_ptr() if keep_slope else base + need, base, need, stream_handle(dev))
    if status:
        raise_for_status(status, "iqk_route_balanced")
    return indices, weights, loss, counts, slope


def route_backward(rows: torch.Tensor, mask, offsets, top_k: int, scoring: int,
                   renormalize: bool, scale: float, indices, grad_weights, slope,
                   grad_loss) -> torch.Tensor:
    """``iqk_route_backward``: the logits' gradient ``[tokens, experts]``."""
    tokens, experts = rows.shape
    if grad_weights is not None:
        grad_weights = grad_weights.to(torch.float32).contiguous()
    if grad_loss is not None:
        grad_loss = grad_loss.to(torch.float32).contiguous()
    grad = rows.new_empty((tokens, experts))
    status = library().iqk_route_backward(
        rows.data_ptr(), DTYPE_IDS[rows.dtype], tokens, experts, rows.stride(0), _ptr(mask),
        _ptr(offsets), 1 if offsets is None else offsets.numel() - 1, top_k, scoring, renormalize,
        scale, indices.data_ptr(), _ptr(grad_weights), _ptr(slope), _ptr(grad_loss),
        grad.data_ptr(), stream_handle(rows.device))
    if status:
        raise_for_status(status, "iqk_route_backward")
    return grad


def mx_quantize(x: torch.Tensor, rows: int, row_stride: int, codes: torch.Tensor,
                scales: torch.Tensor, scale_stride: int) -> None:
    """``iqk_mx_quantize``: ``rows`` rows of ``x``, ``row_stride`` elements apart."""
    status = library().iqk_mx_quantize(
        x.data_ptr(), DTYPE_IDS[x.dtype], rows, x.shape[-1], row_stride, codes.data_ptr(),
        scales.data_ptr(), scale_stride, stream_handle(x.device))
    if status:
        raise_for_status(status, "iqk_mx_quantize")


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, scale_stride: int,
                  out: torch.Tensor) -> None:
    """``iqk_mx_dequantize`` into ``out [..., width]``."""
    width = out.shape[-1]
    status = library().iqk_mx_dequantize(
        codes.data_ptr(), scales.data_ptr(), scale_stride, out.numel() // width, width,
        out.data_ptr(), DTYPE_IDS[out.dtype], stream_handle(out.device))
    if status:
        raise_for_status(status, "iqk_mx_dequantize")


@functools.lru_cache(maxsize=1024)
def mx_workspace_bytes(pairs: int, num_experts: int, width: int, out_features: int) -> int:
    return int(library().iqk_mx_workspace_bytes(pairs, num_experts, width, out_features))


@functools.lru_cache(maxsize=4096)
def mx_few_fits(pairs: int, num_experts: int, out_features: int, width: int, routed: bool) -> bool:
    return bool(library().iqk_mx_few_fits(pairs, num_experts, out_features, width, routed))


_FEW_STATES: dict[tuple[int, int], torch.Tensor] = {}


def mx_few_state(device: torch.device, stream: int, width: int) -> torch.Tensor:
    """Zeroed state of the one-launch product, kept per device and stream (stream
    order keeps a call after the one before). Under graph capture a fresh one of
    what the call uses; where it counts parts, its clearing is part of the graph."""
    if torch.cuda.is_current_stream_capturing():
        need = int(library().iqk_mx_few_state_bytes_for(width))
        state = torch.empty(need, dtype=torch.uint8, device=device)
        if need > 8192:
            state[:8192].zero_()
        return state
    state = _FEW_STATES.get((device.index, stream))
    if state is None:
        state = torch.empty(int(library().iqk_mx_few_state_bytes()), dtype=torch.uint8,
                            device=device)
        state[:8192].zero_()
        if len(_FEW_STATES) >= 64:
            _FEW_STATES.clear()
        _FEW_STATES[device.index, stream] = state
    return state


def mx_few(x: torch.Tensor, rows: int, row_stride: int, sel, pairs: int, codes: torch.Tensor,
           scales: torch.Tensor, scale_stride: int, experts: int, out_features: int,
           y: torch.Tensor) -> None:
    """``iqk_mx_few``: the product of few rows; ``sel`` None for one matrix."""
    stream = stream_handle(y.device)
    state = mx_few_state(y.device, stream, x.shape[-1])
    status = library().iqk_mx_few(
        x.data_ptr(), DTYPE_IDS[x.dtype], rows, row_stride, _ptr(sel), pairs, codes.data_ptr(),
        scales.data_ptr(), scale_stride, experts, out_features, x.shape[-1], y.data_ptr(),
        DTYPE_IDS[y.dtype], state.data_ptr(), state.numel(), stream)
    if status:
        raise_for_status(status, "iqk_mx_few")


def mx_linear(x: torch.Tensor, rows: int, row_stride: int, codes: torch.Tensor,
              scales: torch.Tensor, scale_stride: int, y: torch.Tensor) -> None:
    """``iqk_mx_linear``: ``y [rows, out] = q(x) W^T``."""
    width, out_features = x.shape[-1], codes.shape[0]
    if mx_few_fits(rows, 1, out_features, width, False):
        mx_few(x, rows, row_stride, None, rows, codes, scales, scale_stride, 1, out_features, y)
        return
    need = mx_workspace_bytes(rows, 1, width, out_features)
    ws = y.new_empty(need, dtype=torch.uint8)
    status = library().iqk_mx_linear(
        x.data_ptr(), DTYPE_IDS[x.dtype], rows, row_stride, codes.data_ptr(), scales.data_ptr(),
        scale_stride, out_features, width, y.data_ptr(), DTYPE_IDS[y.dtype], ws.data_ptr(), need,
        stream_handle(y.device))
    if status:
        raise_for_status(status, "iqk_mx_linear")


def check_mx_workspace(workspace: torch.Tensor, device: torch.device | None = None) -> None:
    """A caller's workspace reaches the kernels as an address: refuse what is not
    contiguous bytes on the GPU (on ``device``, where given)."""
    if not isinstance(workspace, torch.Tensor) or workspace.dtype != torch.uint8 \
            or not workspace.is_cuda or not workspace.is_contiguous() \
            or (device is not None and workspace.device != device):
        raise IqkRuntimeError("workspace must be a contiguous uint8 tensor beside the activations")


def mx_routed(x: torch.Tensor, rows: int, row_stride: int, sel: torch.Tensor,
              codes: torch.Tensor, scales: torch.Tensor, scale_stride: int, y: torch.Tensor,
              workspace: torch.Tensor | None = None) -> None:
    """``iqk_mx_routed``: ``y [pairs, out]`` through the stacked matrices."""
    if workspace is not None:
        check_mx_workspace(workspace, y.device)
    pairs, width = sel.numel(), x.shape[-1]
    experts, out_features = codes.shape[0], codes.shape[1]
    if workspace is None:
        if mx_few_fits(pairs, experts, out_features, width, True):
            mx_few(x, rows, row_stride, sel, pairs, codes, scales, scale_stride, experts,
                   out_features, y)
            return
        need = mx_workspace_bytes(pairs, experts, width, out_features)
        workspace = y.new_empty(need, dtype=torch.uint8)
    status = library().iqk_mx_routed(
        x.data_ptr(), DTYPE_IDS[x.dtype], rows, row_stride, sel.data_ptr(), pairs,
        codes.data_ptr(), scales.data_ptr(), scale_stride, experts, out_features, width,
        y.data_ptr(), DTYPE_IDS[y.dtype], workspace.data_ptr(), workspace.numel(),
        stream_handle(y.device))
    if status:
        raise_for_status(status, "iqk_mx_routed")


def mx_set_error(workspace: torch.Tensor, device: torch.device, stray: torch.Tensor) -> None:
    """The error word of a routed call that launched no product: whether an index was
    ``stray``, as ``iqk_mx_routed`` leaves it."""
    check_mx_workspace(workspace, device)
    if workspace.numel() < 16 or workspace.data_ptr() % 16:
        raise IqkRuntimeError("workspace must hold an error word on a 16-byte boundary")
    words = workspace[:16].view(torch.int32)
    words.zero_()
    words[0] = stray * DEVERR_EXPERT


def mx_read_error(workspace: torch.Tensor) -> int:
    """``iqk_mx_read_error``: the device error bits of a routed product's workspace."""
    check_mx_workspace(workspace)
    if workspace.numel() < 16:
        raise IqkRuntimeError("workspace is no routed product's: it has no error word")
    flags = ctypes.c_int32(0)
    raise_for_status(library().iqk_mx_read_error(workspace.data_ptr(), ctypes.byref(flags),
                                                 stream_handle(workspace.device)),
                     "iqk_mx_read_error")
    return int(flags.value)


def mx_take_errors(device: torch.device) -> int:
    """``iqk_mx_take_errors``: the error bits that MXFP4 products left on ``device`` since
    this was last asked (synchronises the current stream). After an error the states of
    the one-launch products start anew."""
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    check_current(device)
    flags = ctypes.c_int32(0)
    raise_for_status(library().iqk_mx_take_errors(ctypes.byref(flags), stream_handle(device)),
                     "iqk_mx_take_errors")
    if flags.value:
        for key in [k for k in _FEW_STATES if k[0] == device.index]:
            del _FEW_STATES[key]
    return int(flags.value)


def read_error(workspace: torch.Tensor, in_features: int, x_rows: int, pairs: int) -> int:
    flags = ctypes.c_int32(0)
    raise_for_status(library().iqk_read_error(workspace.data_ptr(), in_features, x_rows, pairs,
                                              ctypes.byref(flags),
                                              stream_handle(workspace.device)),
                     "iqk_read_error")
    return int(flags.value)


__all__ = [
    "IQ2_MEMBERS", "ROWS_PER_TG", "SUPPORTED_IN_FEATURES", "IqkKernelError", "IqkRuntimeError",
    "check_dequant_geometry", "check_gemv_geometry", "dequant", "gemv", "library",
]
