"""Python binding of libtrellis_sparse.so, the MI355X sparse-voxel conv library.

The library's interface is the C ABI declared in include/trellis_sparse.h; this module loads
it with ctypes and wraps each entry point for torch device tensors (torch supplies device
memory and the current HIP stream; all compute happens in the library's HIP kernels).

There is no fallback: if the shared library is missing or a call fails, an exception is
raised.
"""
from __future__ import annotations

import ctypes
import os
import subprocess
from typing import Any, NamedTuple

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libtrellis_sparse.so")

TSP_F32, TSP_F16, TSP_BF16, TSP_MX8, TSP_KV_MX4 = 0, 1, 2, 3, 4
ALGO = {"auto": 0, "mfma": 1, "narrow": 2, "mfma_gather": 3, "thin": 4, "thin_mfma": 5, "f32_mfma": 6}
STATUS = {0: "OK", 1: "INVALID", 2: "HIP", 3: "RANGE", 4: "UNSUPPORTED", 5: "WORKSPACE"}

# Every extern "C" entry point the header declares (checked by the CPU test suite).
EXPORTS = (
    "tsp_last_error", "tsp_version",
    "tsp_rulebook_workspace_bytes", "tsp_rulebook_build", "tsp_rulebook_build_planned", "tsp_rulebook_count_pairs",
    "tsp_convnext_mlp_packed_bytes", "tsp_convnext_mlp_pack", "tsp_convnext_mlp",
    "tsp_subm_conv3x3", "tsp_subm_conv3x3_ex",
    "tsp_conv_plan_bytes", "tsp_conv_plan_build", "tsp_conv_plan_build_ordered",
    "tsp_conv_weight_pack", "tsp_conv_weight_packed_bytes", "tsp_subm_conv3x3_planned_ln",
    "tsp_subm_conv3x3_planned", "tsp_subm_conv3x3_planned_ex", "tsp_subm_conv3x3_planned_octants",
    "tsp_subm_conv3x3_planned_skip",
    "tsp_subdivide_workspace_bytes", "tsp_subdivide", "tsp_subdivide_noalloc",
    "tsp_linear", "tsp_linear_ex", "tsp_linear_rows_per_call", "tsp_layer_norm", "tsp_c2s_gather", "tsp_c2s_skip_add",
    "tsp_mask_positive",
    "tsp_convnext_workspace_bytes", "tsp_convnext", "tsp_convnext_ex", "tsp_c2s_workspace_bytes", "tsp_c2s",
    "tsp_c2s_ex", "tsp_c2s_part",
    "tsp_group_norm_workspace_bytes", "tsp_group_norm", "tsp_rope_axes", "tsp_attention_workspace_bytes", "tsp_attention",
    "tsp_rms_norm", "tsp_mx_quantize", "tsp_linear_mx_workspace_bytes", "tsp_linear_mx",
    "tsp_kv_page_bytes", "tsp_kv_append", "tsp_kv_gather", "tsp_attention_cached_workspace_bytes", "tsp_attention_cached",
)

BLOCK_CAST_F32 = 2


class ConvNextWeights(ctypes.Structure):
    """tsp_convnext_weights: device pointers, dtypes as tsp_dtype codes."""
    _fields_ = [("conv_weight", ctypes.c_void_p), ("conv_dtype", ctypes.c_int), ("conv_bias", ctypes.c_void_p),
                ("conv_packed", ctypes.c_void_p), ("norm_weight", ctypes.c_void_p),
                ("norm_bias", ctypes.c_void_p), ("mlp0_weight", ctypes.c_void_p), ("mlp0_dtype", ctypes.c_int),
                ("mlp0_bias", ctypes.c_void_p), ("mlp2_weight", ctypes.c_void_p), ("mlp2_dtype", ctypes.c_int),
                ("mlp2_bias", ctypes.c_void_p), ("mlp_packed", ctypes.c_void_p)]


class C2SWeights(ctypes.Structure):
    """tsp_c2s_weights: device pointers, dtypes as tsp_dtype codes."""
    _fields_ = [("norm1_weight", ctypes.c_void_p), ("norm1_bias", ctypes.c_void_p),
                ("conv1_weight", ctypes.c_void_p), ("conv1_dtype", ctypes.c_int), ("conv1_bias", ctypes.c_void_p),
                ("conv1_packed", ctypes.c_void_p), ("conv2_weight", ctypes.c_void_p), ("conv2_dtype", ctypes.c_int),
                ("conv2_bias", ctypes.c_void_p), ("conv2_packed", ctypes.c_void_p)]


class Heads(ctypes.Structure):
    """tsp_heads: rows of heads, strides in elements."""
    _fields_ = [("data", ctypes.c_void_p), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class KvCacheArg(ctypes.Structure):
    """tsp_kv_cache."""
    _fields_ = [("data", ctypes.c_void_p), ("pages", ctypes.c_int64), ("page", ctypes.c_int), ("heads", ctypes.c_int),
                ("d", ctypes.c_int), ("format", ctypes.c_int)]


class TspError(RuntimeError):
    def __init__(self, fn: str, code: int, msg: str):
        super().__init__(f"{fn} -> {STATUS.get(code, code)}: {msg}")
        self.code = code


_lib = None


def build(jobs: int = 8) -> str:
    """Compile libtrellis_sparse.so for gfx950 (hipcc through trellis.cpp_amd/Makefile)."""
    subprocess.run(["make", "-s", "-C", HERE, f"-j{jobs}"], check=True)
    return LIB_PATH


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise FileNotFoundError(
            f"{LIB_PATH} is not built; run `make -C {HERE}` (or __graft_entry__.build())")
    L = ctypes.CDLL(LIB_PATH)
    c_i64, c_int, c_sz, c_vp = ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p
    L.tsp_last_error.restype = ctypes.c_char_p
    L.tsp_last_error.argtypes = []
    L.tsp_version.restype = c_int
    L.tsp_rulebook_workspace_bytes.restype = c_sz
    L.tsp_rulebook_workspace_bytes.argtypes = [c_i64]
    L.tsp_rulebook_build.restype = c_int
    L.tsp_rulebook_build.argtypes = [c_vp, c_i64, c_vp, c_vp, c_sz, c_vp, c_vp]
    L.tsp_convnext_mlp_packed_bytes.restype = c_sz
    L.tsp_convnext_mlp_packed_bytes.argtypes = [c_int]
    L.tsp_convnext_mlp_pack.restype = c_int
    L.tsp_convnext_mlp_pack.argtypes = [c_vp, c_vp, c_int, c_int, c_vp, c_vp]
    L.tsp_convnext_mlp.restype = c_int
    L.tsp_convnext_mlp.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]
    L.tsp_rulebook_build_planned.restype = c_int
    L.tsp_rulebook_build_planned.argtypes = [c_vp, c_i64, c_vp, c_vp, c_sz, c_vp, c_vp, c_sz, c_vp]
    L.tsp_rulebook_count_pairs.restype = c_int
    L.tsp_rulebook_count_pairs.argtypes = [c_vp, c_i64, c_vp, c_vp]
    L.tsp_subm_conv3x3.restype = c_int
    L.tsp_subm_conv3x3.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_int, c_vp, c_int,
                                   c_vp, c_int, c_int, c_vp]
    L.tsp_subm_conv3x3_ex.restype = c_int
    L.tsp_subm_conv3x3_ex.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_int, c_vp, c_int,
                                      c_vp, c_int, c_int, c_int, c_vp, c_vp]
    L.tsp_conv_plan_bytes.restype = c_sz
    L.tsp_conv_plan_bytes.argtypes = [c_i64]
    L.tsp_conv_plan_build.restype = c_int
    L.tsp_conv_plan_build.argtypes = [c_vp, c_i64, c_vp, c_sz, c_vp]
    L.tsp_conv_plan_build_ordered.restype = c_int
    L.tsp_conv_plan_build_ordered.argtypes = [c_vp, c_vp, c_i64, c_vp, c_sz, c_vp]
    L.tsp_conv_weight_pack.restype = c_int
    L.tsp_conv_weight_pack.argtypes = [c_vp, c_int, c_int, c_int, c_vp, c_vp]
    L.tsp_conv_weight_packed_bytes.restype = c_sz
    L.tsp_conv_weight_packed_bytes.argtypes = [c_int, c_int]
    L.tsp_subm_conv3x3_planned_ln.restype = c_int
    L.tsp_subm_conv3x3_planned_ln.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_vp, c_vp, c_int, c_vp, c_vp,
                                              ctypes.c_float, c_vp, c_vp, c_vp]
    L.tsp_subm_conv3x3_planned.restype = c_int
    L.tsp_subm_conv3x3_planned.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_vp, c_vp,
                                           c_int, c_vp, c_int, c_vp]
    L.tsp_subm_conv3x3_planned_ex.restype = c_int
    L.tsp_subm_conv3x3_planned_ex.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_vp, c_vp,
                                              c_int, c_vp, c_int, c_int, c_vp, c_vp]
    L.tsp_subm_conv3x3_planned_octants.restype = c_int
    L.tsp_subm_conv3x3_planned_octants.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_vp,
                                                   c_vp, c_int, c_vp, c_vp, c_vp, c_vp]
    L.tsp_subm_conv3x3_planned_skip.restype = c_int
    L.tsp_subm_conv3x3_planned_skip.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_vp, c_vp,
                                                c_int, c_vp, c_int, c_vp, c_vp, c_vp]
    L.tsp_linear.restype = c_int
    L.tsp_linear.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_int, c_vp, c_int, c_vp, c_int,
                             c_vp]
    L.tsp_linear_ex.restype = c_int
    L.tsp_linear_ex.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_int, c_vp, c_int, c_int, c_vp,
                                c_vp, c_int, c_vp]
    L.tsp_linear_rows_per_call.restype = c_i64
    L.tsp_linear_rows_per_call.argtypes = [c_int, c_int, c_int, c_int, c_int]
    L.tsp_layer_norm.restype = c_int
    L.tsp_layer_norm.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, ctypes.c_float, c_int,
                                 c_vp, c_int, c_vp]
    L.tsp_c2s_gather.restype = c_int
    L.tsp_c2s_gather.argtypes = [c_vp, c_int, c_vp, c_i64, c_int, c_vp, c_vp]
    L.tsp_c2s_skip_add.restype = c_int
    L.tsp_c2s_skip_add.argtypes = [c_vp, c_int, c_vp, c_i64, c_int, c_int, c_vp, c_int, c_vp]
    L.tsp_mask_positive.restype = c_int
    L.tsp_mask_positive.argtypes = [c_vp, c_i64, c_vp, c_vp]
    L.tsp_subdivide_workspace_bytes.restype = c_sz
    L.tsp_subdivide_workspace_bytes.argtypes = [c_i64]
    L.tsp_subdivide.restype = c_int
    L.tsp_subdivide.argtypes = [c_vp, c_vp, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_sz, c_vp]
    L.tsp_subdivide_noalloc.restype = c_int
    L.tsp_subdivide_noalloc.argtypes = [c_vp, c_vp, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp]
    cnw, c2w = ctypes.POINTER(ConvNextWeights), ctypes.POINTER(C2SWeights)
    L.tsp_convnext_workspace_bytes.restype = c_sz
    L.tsp_convnext_workspace_bytes.argtypes = [c_i64, c_int, c_int, cnw, c_int, c_int]
    L.tsp_convnext.restype = c_int
    L.tsp_convnext.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, cnw, c_vp, c_vp, c_sz, c_int, c_vp]
    L.tsp_convnext_ex.restype = c_int
    L.tsp_convnext_ex.argtypes = [c_vp, c_int, c_vp, c_i64, c_int, c_vp, c_vp, cnw, c_vp, c_vp, c_int, c_vp, c_sz,
                                  c_int, c_vp]
    L.tsp_c2s_workspace_bytes.restype = c_sz
    L.tsp_c2s_workspace_bytes.argtypes = [c_i64, c_i64, c_int, c_int, c2w, c_int, c_int, c_int]
    L.tsp_c2s.restype = c_int
    L.tsp_c2s.argtypes = [c_vp, c_i64, c_int, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_int, c_vp, c_vp, c2w,
                          c_vp, c_vp, c_sz, c_int, c_vp]
    L.tsp_c2s_ex.restype = c_int
    L.tsp_c2s_ex.argtypes = [c_vp, c_i64, c_int, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_int, c_vp, c_vp, c2w,
                             c_vp, c_vp, c_int, c_vp, c_sz, c_int, c_vp]
    L.tsp_c2s_part.restype = c_int
    L.tsp_c2s_part.argtypes = [c_vp, c_i64, c_int, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_int, c_vp, c_vp, c2w,
                               c_vp, c_vp, c_int, c_vp, c_sz, c_int, c_int, c_i64, c_i64, c_vp]
    c_f, hp = ctypes.c_float, ctypes.POINTER(Heads)
    L.tsp_group_norm_workspace_bytes.restype = c_sz
    L.tsp_group_norm_workspace_bytes.argtypes = [c_i64, c_int, c_int, c_int]
    L.tsp_group_norm.restype = c_int
    L.tsp_group_norm.argtypes = [c_vp, c_int, c_i64, c_int, c_int, c_vp, c_int, c_vp, c_vp, c_f, c_int, c_vp, c_int, c_vp,
                                 c_sz, c_vp]
    L.tsp_rope_axes.restype = c_int
    L.tsp_rope_axes.argtypes = [hp, c_int, hp, c_int, c_int, c_i64, c_int, c_vp, c_int, ctypes.POINTER(c_int),
                                ctypes.c_double, c_int, c_vp, c_vp, c_f, hp, hp, c_int, c_vp]
    L.tsp_attention_workspace_bytes.restype = c_sz
    L.tsp_attention_workspace_bytes.argtypes = [c_i64, c_i64, c_int, c_int, c_int, c_int]
    L.tsp_attention.restype = c_int
    L.tsp_attention.argtypes = [hp, hp, hp, c_int, c_i64, c_i64, c_int, c_int, c_int, c_vp, c_vp, c_int, c_f, c_int, hp,
                                c_vp, c_sz, c_vp]
    L.tsp_rms_norm.restype = c_int
    L.tsp_rms_norm.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_int, c_vp, c_f, c_vp, c_int, c_vp, c_vp, c_vp]
    L.tsp_mx_quantize.restype = c_int
    L.tsp_mx_quantize.argtypes = [c_vp, c_int, c_i64, c_int, c_vp, c_vp, c_vp]
    L.tsp_linear_mx_workspace_bytes.restype = c_sz
    L.tsp_linear_mx_workspace_bytes.argtypes = [c_i64, c_int, c_int]
    L.tsp_linear_mx.restype = c_int
    L.tsp_linear_mx.argtypes = [c_vp, c_vp, c_i64, c_int, c_vp, c_vp, c_vp, c_int, c_int, c_vp, c_vp, c_int, c_vp, c_sz, c_vp]
    kvp = ctypes.POINTER(KvCacheArg)
    L.tsp_kv_page_bytes.restype = c_sz
    L.tsp_kv_page_bytes.argtypes = [c_int, c_int, c_int, c_int]
    L.tsp_kv_append.restype = c_int
    L.tsp_kv_append.argtypes = [kvp, hp, hp, c_int, c_i64, c_vp, c_int, c_vp, c_int, c_vp, hp, c_int, c_vp, c_int,
                                ctypes.POINTER(c_int), ctypes.c_double, c_int, c_vp, c_vp, ctypes.c_double, hp, c_vp]
    L.tsp_kv_gather.restype = c_int
    L.tsp_kv_gather.argtypes = [kvp, c_i64, c_vp, c_int, c_vp, c_int, c_vp, hp, hp, c_int, c_vp]
    L.tsp_attention_cached_workspace_bytes.restype = c_sz
    L.tsp_attention_cached_workspace_bytes.argtypes = [c_i64, c_int, c_int, kvp, c_int]
    L.tsp_attention_cached.restype = c_int
    L.tsp_attention_cached.argtypes = [hp, c_int, c_i64, c_int, kvp, c_vp, c_int, c_vp, c_int, c_vp, c_f, c_int, hp, c_vp, c_sz,
                                       c_vp]
    _lib = L
    return L


def _check(fn: str, code: int) -> None:
    if code != 0:
        raise TspError(fn, code, lib().tsp_last_error().decode(errors="replace"))


# --------------------------------------------------------------------------------------------
# torch conveniences (device memory + stream plumbing only)
# --------------------------------------------------------------------------------------------
def _torch():
    import torch
    return torch


_codes = {}


def dtype_code(dt) -> int:
    if not _codes:
        torch = _torch()
        _codes.update({torch.float32: TSP_F32, torch.float16: TSP_F16, torch.bfloat16: TSP_BF16})
    return _codes[dt]


def _stream(stream=None):
    torch = _torch()
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("tensors must live on the GPU")


def _table_buffers(c, n, nbr, workspace):
    torch = _torch()
    ws_bytes = lib().tsp_rulebook_workspace_bytes(n)
    if nbr is None:
        nbr = torch.empty(27 * n, dtype=torch.int32, device=c.device)
    elif nbr.dtype != torch.int32 or nbr.numel() != 27 * n or not nbr.is_contiguous():
        raise ValueError("nbr must be a contiguous int32 buffer of 27*N")
    if workspace is None:
        workspace = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=c.device)
    elif workspace.dtype != torch.uint8 or workspace.numel() < ws_bytes:
        raise ValueError("workspace must be a uint8 buffer of tsp_rulebook_workspace_bytes(N)")
    return nbr, workspace, ws_bytes


def rulebook_build(coords, check: bool = True, nbr=None, workspace=None, stream=None):
    """coords int32 [N,3] on the GPU -> tap-major int32 neighbour table [27*N] (sentinel N).
    nbr and workspace (uint8, tsp_rulebook_workspace_bytes(N)) may be given to reuse buffers;
    check=False skips the range check's read-back."""
    torch = _torch()
    _require_cuda(coords)
    c = coords.contiguous()
    if c.dtype != torch.int32 or c.dim() != 2 or c.shape[1] != 3:
        raise ValueError("coords must be int32 [N, 3]")
    n = c.shape[0]
    nbr, ws, ws_bytes = _table_buffers(c, n, nbr, workspace)
    status = torch.zeros(1, dtype=torch.int32, device=c.device) if check else None
    _check("tsp_rulebook_build",
           lib().tsp_rulebook_build(_ptr(c), n, _ptr(nbr), _ptr(ws), ws_bytes, _ptr(status),
                                    _stream(stream)))
    if check and n and int(status.item()) != 0:
        raise TspError("tsp_rulebook_build", 3, "coordinate outside [0, 2^21-3]")
    return nbr


def rulebook_build_planned(coords, check: bool = True, nbr=None, workspace=None, plan=None, stream=None):
    """coords int32 [N,3] on the GPU -> (neighbour table int32 [27*N], Morton-ordered conv plan
    uint8 buffer): rulebook_build and conv_plan_build(coords=...) in one call on one cell grid.
    nbr, workspace (uint8, tsp_rulebook_workspace_bytes(N)) and plan (uint8, tsp_conv_plan_bytes(N))
    may be given to reuse buffers."""
    torch = _torch()
    _require_cuda(coords)
    c = coords.contiguous()
    if c.dtype != torch.int32 or c.dim() != 2 or c.shape[1] != 3:
        raise ValueError("coords must be int32 [N, 3]")
    n = c.shape[0]
    nbr, workspace, ws_bytes = _table_buffers(c, n, nbr, workspace)
    nb = lib().tsp_conv_plan_bytes(n)
    if plan is None:
        plan = torch.empty(max(nb, 1), dtype=torch.uint8, device=c.device)
    elif plan.dtype != torch.uint8 or plan.numel() < nb:
        raise ValueError("plan must be a uint8 buffer of tsp_conv_plan_bytes(N)")
    status = torch.zeros(1, dtype=torch.int32, device=c.device) if check else None
    _check("tsp_rulebook_build_planned",
           lib().tsp_rulebook_build_planned(_ptr(c), n, _ptr(nbr), _ptr(workspace), ws_bytes,
                                            _ptr(status), _ptr(plan), nb,
                                            _stream(stream)))
    if check and n and int(status.item()) != 0:
        raise TspError("tsp_rulebook_build_planned", 3, "coordinate outside [0, 2^21-3]")
    return nbr, plan


def convnext_mlp_pack(w0, w2, stream=None):
    """w0 [4C, C], w2 [C, 4C] of one 16-bit dtype -> the packed buffer tsp_convnext_mlp reads."""
    torch = _torch()
    _require_cuda(w0, w2)
    c = w0.shape[1]
    if w2.dtype != w0.dtype or tuple(w0.shape) != (4 * c, c) or tuple(w2.shape) != (c, 4 * c):
        raise ValueError("w0 [4C, C] and w2 [C, 4C] of one dtype")
    w0, w2 = w0.contiguous(), w2.contiguous()
    packed = torch.empty(lib().tsp_convnext_mlp_packed_bytes(c) // 2, dtype=w0.dtype, device=w0.device)
    _check("tsp_convnext_mlp_pack",
           lib().tsp_convnext_mlp_pack(_ptr(w0), _ptr(w2), dtype_code(w0.dtype), c, _ptr(packed), _stream(stream)))
    return packed


def convnext_mlp(xn, packed, b0, b2, x, out=None, stream=None):
    """The ConvNeXt MLP in one kernel: out f32 [N, C] = x + b2 + w2 . silu(w0 . xn + b0) for xn
    [N, C] (16-bit), the weights packed by convnext_mlp_pack, x f32 [N, C], C = 128; out may be x."""
    torch = _torch()
    _require_cuda(xn, packed, x)
    n, c = xn.shape
    if packed.dtype != xn.dtype or packed.numel() * 2 != lib().tsp_convnext_mlp_packed_bytes(c):
        raise ValueError("packed must come from convnext_mlp_pack with xn's dtype and C")
    if x.dtype != torch.float32 or tuple(x.shape) != (n, c):
        raise ValueError("x must be float32 [N, C]")
    for name, b, size in (("b0", b0, 4 * c), ("b2", b2, c)):
        if b is not None and (b.dtype != torch.float32 or b.numel() != size or not b.is_contiguous()
                              or b.device != xn.device):
            raise ValueError(f"{name} must be a contiguous float32 vector of {size} on xn's device")
    if out is None:
        out = torch.empty((n, c), dtype=torch.float32, device=xn.device)
    elif (out.dtype != torch.float32 or tuple(out.shape) != (n, c) or not out.is_contiguous()
          or out.device != xn.device):
        raise ValueError("out must be a contiguous float32 [N, C] tensor on xn's device")
    xn, x = xn.contiguous(), x.contiguous()
    _check("tsp_convnext_mlp",
           lib().tsp_convnext_mlp(_ptr(xn), dtype_code(xn.dtype), n, c, _ptr(packed), _ptr(b0), _ptr(b2),
                                  _ptr(x), _ptr(out), _stream(stream)))
    return out


def count_pairs(nbr, n: int, stream=None) -> int:
    torch = _torch()
    _require_cuda(nbr)
    cnt = torch.zeros(1, dtype=torch.int64, device=nbr.device)
    _check("tsp_rulebook_count_pairs",
           lib().tsp_rulebook_count_pairs(_ptr(nbr), n, _ptr(cnt), _stream(stream)))
    return int(cnt.item())


def _check_out(out, n: int, co: int, dtype, device):
    """A caller's out= must be a contiguous [n, co] tensor of the output dtype on the device the
    inputs are on: the kernels write n * co elements through its raw pointer."""
    if tuple(out.shape) != (n, co):
        raise ValueError(f"out must have shape ({n}, {co}), got {tuple(out.shape)}")
    if out.dtype != dtype:
        raise ValueError(f"out must be {dtype}, got {out.dtype}")
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    if out.device != device:
        raise ValueError(f"out must live on {device}, got {out.device}")


def _f32_vec(t, n: int, name: str):
    """An optional float32 vector of at least n elements: the kernels read n through its pointer."""
    if t is None:
        return None
    if t.dtype != _torch().float32 or t.numel() < n:
        raise ValueError(f"{name} must be float32 with {n} elements")
    return t.contiguous()


def _check_nbr(nbr, n: int, device):
    torch = _torch()
    if nbr.dtype != torch.int32 or nbr.numel() != 27 * n or not nbr.is_contiguous():
        raise ValueError(f"nbr must be a contiguous int32 table of 27*N = {27 * n} entries")
    if nbr.device != device:
        raise ValueError("nbr must live on the features' device")


def subm_conv3x3(feats, nbr, weight, bias, out_dtype=None, algo: str = "auto", out=None,
                 zero_pad: bool = False, row0=None, stream=None):
    """feats [N,Ci], nbr int32 [27*N], weight [Co,27,Ci], bias f32 [Co] -> out [N,Co].
    zero_pad: absent taps read an exact zero row instead of 0 * feats[0]; row0 (float32 [Ci]):
    the unrounded row 0 the features were rounded from, whose 0 * row0 is the padding row."""
    torch = _torch()
    if feats.dim() != 2:
        raise ValueError("feats must be [N, Ci]")
    n, ci = feats.shape
    co = weight.shape[0]
    if weight.shape != (co, 27, ci):
        raise ValueError(f"weight must be [Co,27,Ci]=[{co},27,{ci}], got {tuple(weight.shape)}")
    _check_nbr(nbr, n, feats.device)
    if bias.dtype != torch.float32 or bias.numel() != co:
        raise ValueError("bias must be float32 [Co]")
    if row0 is not None and (row0.dtype != torch.float32 or row0.numel() != ci):
        raise ValueError("row0 must be float32 [Ci]")
    odt = out_dtype or feats.dtype
    if out is None:
        out = torch.empty((n, co), dtype=odt, device=feats.device)
    else:
        _check_out(out, n, co, odt, feats.device)
    _require_cuda(feats, nbr, weight, bias, out, row0)
    f, w, b = feats.contiguous(), weight.contiguous(), bias.contiguous()
    r0 = row0.contiguous() if row0 is not None else None
    _check("tsp_subm_conv3x3_ex",
           lib().tsp_subm_conv3x3_ex(_ptr(f), dtype_code(f.dtype), n, ci, _ptr(nbr), _ptr(w),
                                     dtype_code(w.dtype), _ptr(b), co, _ptr(out),
                                     dtype_code(out.dtype), ALGO[algo], 1 if zero_pad else 0,
                                     _ptr(r0), _stream(stream)))
    return out


def conv_plan_build(nbr, n: int, coords=None, plan=None, stream=None):
    """Plan of neighbour table nbr (int32 [27*N]) for the planned convs -> uint8 buffer (plan, of
    tsp_conv_plan_bytes(N), may be given to reuse it). With coords (int32 [N, 3], the coordinates
    the table was built from) tiles follow the Morton order of the voxels' 8^3 cells; without,
    tiles are consecutive rows."""
    torch = _torch()
    _require_cuda(nbr, coords)
    _check_nbr(nbr, n, nbr.device)
    nb = lib().tsp_conv_plan_bytes(n)
    if plan is None:
        plan = torch.empty(max(nb, 1), dtype=torch.uint8, device=nbr.device)
    elif plan.dtype != torch.uint8 or plan.numel() < nb:
        raise ValueError("plan must be a uint8 buffer of tsp_conv_plan_bytes(N)")
    if coords is None:
        _check("tsp_conv_plan_build",
               lib().tsp_conv_plan_build(_ptr(nbr), n, _ptr(plan), nb, _stream(stream)))
    else:
        c = coords.contiguous()
        if c.dtype != torch.int32 or tuple(c.shape) != (n, 3):
            raise ValueError("coords must be int32 [N, 3]")
        _check("tsp_conv_plan_build_ordered",
               lib().tsp_conv_plan_build_ordered(_ptr(nbr), _ptr(c), n, _ptr(plan), nb, _stream(stream)))
    return plan


def conv_weight_pack(weight, stream=None):
    """W [Co,27,Ci] f16/bf16 -> packed copy (same dtype, flat): the values in operand order, then
    the 256-byte trailer (tsp_conv_weight_packed_bytes(Ci, Co) bytes in all)."""
    torch = _torch()
    _require_cuda(weight)
    w = weight.contiguous()
    co, _, ci = w.shape
    packed = torch.empty(lib().tsp_conv_weight_packed_bytes(ci, co) // 2, dtype=w.dtype, device=w.device)
    _check("tsp_conv_weight_pack",
           lib().tsp_conv_weight_pack(_ptr(w), dtype_code(w.dtype), ci, co, _ptr(packed),
                                      _stream(stream)))
    return packed


def _check_planned(feats, nbr, plan, packed_weight, ci: int, co: int):
    n = feats.shape[0]
    _check_nbr(nbr, n, feats.device)
    need = lib().tsp_conv_plan_bytes(n)
    if plan.numel() * plan.element_size() < need:
        raise ValueError(f"plan holds {plan.numel() * plan.element_size()} bytes; a table of {n} "
                         f"voxels needs {need}")
    if packed_weight.dtype != feats.dtype:
        raise ValueError(f"packed weight is {packed_weight.dtype}, features are {feats.dtype}")
    if packed_weight.numel() * packed_weight.element_size() != lib().tsp_conv_weight_packed_bytes(ci, co):
        raise ValueError("packed weight size does not match [Co,27,Ci] (see conv_weight_pack)")
    if not packed_weight.is_contiguous():
        raise ValueError("packed weight must be contiguous")


def subm_conv3x3_planned(feats, nbr, plan, packed_weight, bias, co: int, out_dtype=None, out=None,
                         zero_pad: bool = False, row0=None, stream=None):
    """The MFMA conv with a plan (conv_plan_build) and packed weights (conv_weight_pack).
    zero_pad: absent taps read an exact zero row; row0 (float32 [Ci]): the unrounded row 0 the
    features were rounded from, whose 0 * row0 is the padding row."""
    torch = _torch()
    if feats.dim() != 2:
        raise ValueError("feats must be [N, Ci]")
    n, ci = feats.shape
    _check_planned(feats, nbr, plan, packed_weight, ci, co)
    if bias.dtype != torch.float32 or bias.numel() != co:
        raise ValueError("bias must be float32 [Co]")
    if row0 is not None and (row0.dtype != torch.float32 or row0.numel() != ci):
        raise ValueError("row0 must be float32 [Ci]")
    odt = out_dtype or feats.dtype
    if out is None:
        out = torch.empty((n, co), dtype=odt, device=feats.device)
    else:
        _check_out(out, n, co, odt, feats.device)
    _require_cuda(feats, nbr, plan, packed_weight, bias, out, row0)
    f = feats.contiguous()
    r0 = row0.contiguous() if row0 is not None else None
    _check("tsp_subm_conv3x3_planned_ex",
           lib().tsp_subm_conv3x3_planned_ex(_ptr(f), dtype_code(f.dtype), n, ci, _ptr(nbr),
                                             _ptr(plan), _ptr(packed_weight), _ptr(bias), co,
                                             _ptr(out), dtype_code(out.dtype),
                                             1 if zero_pad else 0, _ptr(r0), _stream(stream)))
    return out


def subm_conv3x3_planned_ln(feats, nbr, plan, packed_weight, bias, co: int, norm_weight, norm_bias,
                            eps: float = 1e-6, out=None, row0=None, stream=None):
    """The planned conv with each output row layer-normalised by its stores (co = 64 or 128):
    (h - mean) / sqrt(var + eps) * norm_weight + norm_bias for h = conv + bias, in the feature
    dtype."""
    torch = _torch()
    if feats.dim() != 2:
        raise ValueError("feats must be [N, Ci]")
    n, ci = feats.shape
    _check_planned(feats, nbr, plan, packed_weight, ci, co)
    for name, t in (("bias", bias), ("norm_weight", norm_weight), ("norm_bias", norm_bias)):
        if t.dtype != torch.float32 or t.numel() != co:
            raise ValueError(f"{name} must be float32 [Co]")
    if row0 is not None and (row0.dtype != torch.float32 or row0.numel() != ci):
        raise ValueError("row0 must be float32 [Ci]")
    if out is None:
        out = torch.empty((n, co), dtype=feats.dtype, device=feats.device)
    else:
        _check_out(out, n, co, feats.dtype, feats.device)
    _require_cuda(feats, nbr, plan, packed_weight, bias, norm_weight, norm_bias, out, row0)
    f = feats.contiguous()
    r0 = row0.contiguous() if row0 is not None else None
    _check("tsp_subm_conv3x3_planned_ln",
           lib().tsp_subm_conv3x3_planned_ln(_ptr(f), dtype_code(f.dtype), n, ci, _ptr(nbr), _ptr(plan),
                                             _ptr(packed_weight), _ptr(bias), co, _ptr(norm_weight),
                                             _ptr(norm_bias), float(eps), _ptr(out), _ptr(r0), _stream(stream)))
    return out


def subm_conv3x3_planned_octants(feats, nbr, plan, packed_weight, bias, cout: int, mask, mstart,
                                 m: int, stream=None):
    """The C2S conv1 with its octant gather in the stores: the planned conv to 8*cout channels,
    parent i's channels [o*cout, +cout) written to its child of octant o (mask and mstart as
    given to / returned by subdivide) -> float32 [M, cout]."""
    torch = _torch()
    n, ci = feats.shape
    co = 8 * cout
    _check_planned(feats, nbr, plan, packed_weight, ci, co)
    if bias.dtype != torch.float32 or bias.numel() != co:
        raise ValueError("bias must be float32 [8*cout]")
    m8 = mask.reshape(-1).contiguous()
    if m8.dtype != torch.uint8 or m8.numel() != 8 * n:
        raise ValueError("mask must be uint8 with 8*N entries")
    if mstart.dtype != torch.int32 or mstart.numel() != n + 1:
        raise ValueError("mstart must be int32 [N+1]")
    _require_cuda(feats, nbr, plan, packed_weight, bias, mask, mstart)
    # the kernel writes rows up to mstart[N] - 1: the output must hold exactly that many
    if n and int(mstart[-1].item()) != m:
        raise ValueError(f"m={m} but the subdivision has mstart[N]={int(mstart[-1].item())} children")
    out = torch.empty((m, cout), dtype=torch.float32, device=feats.device)
    f = feats.contiguous()
    _check("tsp_subm_conv3x3_planned_octants",
           lib().tsp_subm_conv3x3_planned_octants(_ptr(f), dtype_code(f.dtype), n, ci, _ptr(nbr),
                                                  _ptr(plan), _ptr(packed_weight), _ptr(bias), cout,
                                                  _ptr(m8), _ptr(mstart), _ptr(out),
                                                  _stream(stream)))
    return out


def subm_conv3x3_planned_skip(feats, nbr, plan, packed_weight, bias, co: int, x, gidx, stream=None):
    """The C2S conv2 with the block's skip added by its stores: the planned conv (f32 out) over
    the M children plus repeat_interleave of x's octant blocks (x float32 [N, cin], gidx from
    subdivide) -> float32 [M, co]."""
    torch = _torch()
    m, ci = feats.shape
    _check_planned(feats, nbr, plan, packed_weight, ci, co)
    if bias.dtype != torch.float32 or bias.numel() != co:
        raise ValueError("bias must be float32 [Co]")
    xc = x.contiguous()
    if xc.dtype != torch.float32 or xc.dim() != 2:
        raise ValueError("x must be float32 [N, cin]")
    if gidx.dtype != torch.int32 or gidx.numel() != m:
        raise ValueError("gidx must be int32 [M]")
    _require_cuda(feats, nbr, plan, packed_weight, bias, x, gidx)
    # the stores read x[gidx // 8]: every gidx must name an octant of a row of x
    if m and not (0 <= int(gidx.min().item()) and int(gidx.max().item()) < 8 * xc.shape[0]):
        raise ValueError("gidx holds an octant outside x's rows")
    out = torch.empty((m, co), dtype=torch.float32, device=feats.device)
    f = feats.contiguous()
    _check("tsp_subm_conv3x3_planned_skip",
           lib().tsp_subm_conv3x3_planned_skip(_ptr(f), dtype_code(f.dtype), m, ci, _ptr(nbr),
                                               _ptr(plan), _ptr(packed_weight), _ptr(bias), co,
                                               _ptr(xc), xc.shape[1], _ptr(gidx), _ptr(out),
                                               _stream(stream)))
    return out


def subdivide(mask, coords, stream=None):
    """mask uint8 [8N] (or [N,8]), coords int32 [N,3] -> (child coords [M,3], gidx [M],
    mstart [N+1])."""
    torch = _torch()
    _require_cuda(mask, coords)
    c = coords.contiguous()
    n = c.shape[0]
    m8 = mask.reshape(-1).contiguous()
    if m8.dtype != torch.uint8 or m8.numel() != 8 * n:
        raise ValueError("mask must be uint8 with 8*N entries")
    mstart = torch.empty(n + 1, dtype=torch.int32, device=c.device)
    child = torch.empty((max(8 * n, 1), 3), dtype=torch.int32, device=c.device)
    gidx = torch.empty(max(8 * n, 1), dtype=torch.int32, device=c.device)
    m_dev = torch.empty(1, dtype=torch.int64, device=c.device)
    ws_bytes = lib().tsp_subdivide_workspace_bytes(n)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=c.device)
    _check("tsp_subdivide",
           lib().tsp_subdivide(_ptr(m8), _ptr(c), n, _ptr(mstart), _ptr(child), _ptr(gidx),
                               _ptr(m_dev), _ptr(ws), ws_bytes, _stream(stream)))
    m = int(m_dev.item())
    return child[:m], gidx[:m], mstart


def linear(x, weight, bias=None, out_dtype=None, stream=None):
    """x [N,Ci] . W^T + bias for W [Co,Ci] -> [N,Co] (fp32 accumulation)."""
    torch = _torch()
    bias = _f32_vec(bias, weight.shape[0], "bias")
    _require_cuda(x, weight, bias)
    n, ci = x.shape
    co = weight.shape[0]
    if weight.shape != (co, ci):
        raise ValueError("weight must be [Co, Ci]")
    out = torch.empty((n, co), dtype=out_dtype or x.dtype, device=x.device)
    xc, wc = x.contiguous(), weight.contiguous()
    _check("tsp_linear",
           lib().tsp_linear(_ptr(xc), dtype_code(xc.dtype), n, ci, _ptr(wc), dtype_code(wc.dtype),
                            _ptr(bias), co, _ptr(out), dtype_code(out.dtype), _stream(stream)))
    return out


ACT = {"none": 0, "silu": 1}


def linear_ex(x, weight, bias=None, act: str = "none", residual=None, out_dtype=None, stream=None):
    """act(x [N,Ci] . W^T + bias) + residual for W [Co,Ci] -> [N,Co], one library GEMM with the
    bias, activation and residual in its epilogue (16-bit x and W of one dtype; raises
    TspError UNSUPPORTED otherwise)."""
    torch = _torch()
    bias = _f32_vec(bias, weight.shape[0], "bias")
    _require_cuda(x, weight, bias, residual)
    n, ci = x.shape
    co = weight.shape[0]
    if weight.shape != (co, ci):
        raise ValueError("weight must be [Co, Ci]")
    if residual is not None and (residual.dtype != torch.float32 or residual.shape != (n, co)):
        raise ValueError("residual must be float32 [N, Co]")
    out = torch.empty((n, co), dtype=out_dtype or x.dtype, device=x.device)
    xc, wc = x.contiguous(), weight.contiguous()
    rc = residual.contiguous() if residual is not None else None
    _check("tsp_linear_ex",
           lib().tsp_linear_ex(_ptr(xc), dtype_code(xc.dtype), n, ci, _ptr(wc), dtype_code(wc.dtype),
                               _ptr(bias), co, ACT[act], _ptr(rc), _ptr(out), dtype_code(out.dtype),
                               _stream(stream)))
    return out


def layer_norm(x, gamma=None, beta=None, eps: float = 1e-6, silu: bool = False, out_dtype=None,
               stream=None):
    """Row LayerNorm over channels (biased variance) [* gamma + beta] [then SiLU]."""
    torch = _torch()
    gamma, beta = _f32_vec(gamma, x.shape[1], "gamma"), _f32_vec(beta, x.shape[1], "beta")
    _require_cuda(x, gamma, beta)
    xc = x.contiguous()
    n, c = xc.shape
    out = torch.empty((n, c), dtype=out_dtype or x.dtype, device=x.device)
    _check("tsp_layer_norm",
           lib().tsp_layer_norm(_ptr(xc), dtype_code(xc.dtype), n, c, _ptr(gamma), _ptr(beta),
                                eps, 1 if silu else 0, _ptr(out), dtype_code(out.dtype),
                                _stream(stream)))
    return out


def c2s_gather(h, gidx, cout: int, stream=None):
    """h [N, 8*cout] -> [M, cout]: child m takes block gidx[m] % 8 of parent gidx[m] // 8."""
    torch = _torch()
    _require_cuda(h, gidx)
    m = gidx.numel()
    out = torch.empty((m, cout), dtype=h.dtype, device=h.device)
    hc = h.contiguous()
    _check("tsp_c2s_gather",
           lib().tsp_c2s_gather(_ptr(hc), dtype_code(hc.dtype), _ptr(gidx), m, cout, _ptr(out),
                                _stream(stream)))
    return out


def c2s_skip_add(x, gidx, acc, stream=None):
    """acc [M, Cout] += repeat_interleave(x.reshape(8N, Cin/8)[gidx], Cout/(Cin/8)) in place."""
    _require_cuda(x, gidx, acc)
    xc = x.contiguous()
    m, cout = acc.shape
    _check("tsp_c2s_skip_add",
           lib().tsp_c2s_skip_add(_ptr(xc), dtype_code(xc.dtype), _ptr(gidx), m, xc.shape[1],
                                  cout, _ptr(acc), dtype_code(acc.dtype), _stream(stream)))
    return acc


def mask_positive(logits, stream=None):
    """uint8 mask of logits > 0 (float32 input, any shape)."""
    torch = _torch()
    if logits.dtype != torch.float32:   # (the kernel would read twice a 16-bit tensor's bytes)
        raise ValueError(f"logits must be float32, got {logits.dtype}")
    _require_cuda(logits)
    lc = logits.contiguous()
    mask = torch.empty(lc.shape, dtype=torch.uint8, device=lc.device)
    _check("tsp_mask_positive",
           lib().tsp_mask_positive(_ptr(lc), lc.numel(), _ptr(mask), _stream(stream)))
    return mask


def _vec(t, n: int, name: str):
    torch = _torch()
    if t.dtype != torch.float32 or t.numel() != n:
        raise ValueError(f"{name} must be float32 [{n}]")
    return t.contiguous()


def _mat(t, shape, name: str):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t.contiguous()


def convnext(x, nbr, p: dict, plan=None, cast_f32: bool = False, stream=None, x16=None, out16_dtype=None):
    """SparseConvNeXtBlock3d through tsp_convnext_ex: x [N, C] (f32, or 16-bit of the conv input's
    type), p the block's tensors by their reference names without the prefix ("conv.weight"
    [C,27,C], "conv.bias", "norm.weight", "norm.bias", "mlp.0.weight" [4C,C], "mlp.0.bias",
    "mlp.2.weight" [C,4C], "mlp.2.bias"); optional "conv.packed" (conv_weight_pack) and
    "mlp.packed" (convnext_mlp_pack of mlp.0 and mlp.2). x16, optional with f32 x: x already
    rounded to the conv input's 16-bit type. -> f32 [N, C], or (out, out rounded to out16_dtype)
    when out16_dtype (torch.bfloat16 / torch.float16) is given."""
    torch = _torch()
    n, c = x.shape
    _check_nbr(nbr, n, x.device)
    t = {"conv.weight": _mat(p["conv.weight"], (c, 27, c), "conv.weight"),
         "mlp.0.weight": _mat(p["mlp.0.weight"], (4 * c, c), "mlp.0.weight"),
         "mlp.2.weight": _mat(p["mlp.2.weight"], (c, 4 * c), "mlp.2.weight")}
    for k, m in (("conv.bias", c), ("norm.weight", c), ("norm.bias", c), ("mlp.0.bias", 4 * c), ("mlp.2.bias", c)):
        t[k] = _vec(p[k], m, k)
    packed = p.get("conv.packed")
    if packed is not None and (packed.numel() * packed.element_size() != lib().tsp_conv_weight_packed_bytes(c, c)):
        raise ValueError("conv.packed must be conv.weight packed by conv_weight_pack")
    mpacked = p.get("mlp.packed")
    if mpacked is not None and mpacked.numel() * mpacked.element_size() != lib().tsp_convnext_mlp_packed_bytes(c):
        raise ValueError("mlp.packed must be mlp.0 and mlp.2 packed by convnext_mlp_pack")
    if plan is not None and (plan.dtype != torch.uint8 or plan.numel() < lib().tsp_conv_plan_bytes(n)):
        raise ValueError("plan must be a uint8 buffer of tsp_conv_plan_bytes(N)")
    _require_cuda(x, nbr, plan, packed, mpacked, *t.values())
    w = ConvNextWeights(_ptr(t["conv.weight"]), dtype_code(t["conv.weight"].dtype), _ptr(t["conv.bias"]),
                        _ptr(packed), _ptr(t["norm.weight"]), _ptr(t["norm.bias"]), _ptr(t["mlp.0.weight"]),
                        dtype_code(t["mlp.0.weight"].dtype), _ptr(t["mlp.0.bias"]), _ptr(t["mlp.2.weight"]),
                        dtype_code(t["mlp.2.weight"].dtype), _ptr(t["mlp.2.bias"]), _ptr(mpacked))
    flags = BLOCK_CAST_F32 if cast_f32 else 0
    xc = x.contiguous()
    if x16 is not None:
        x16 = x16.contiguous()
        if tuple(x16.shape) != (n, c) or x16.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("x16 must be a 16-bit [N, C] tensor")
        _require_cuda(x16)
    out = torch.empty((n, c), dtype=torch.float32, device=x.device)
    out16 = None if out16_dtype is None else torch.empty((n, c), dtype=out16_dtype, device=x.device)
    nb = lib().tsp_convnext_workspace_bytes(n, c, dtype_code(xc.dtype), ctypes.byref(w), int(plan is not None), flags)
    ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=x.device)
    _check("tsp_convnext_ex", lib().tsp_convnext_ex(
        _ptr(xc), dtype_code(xc.dtype), _ptr(x16), n, c, _ptr(nbr), _ptr(plan), ctypes.byref(w), _ptr(out),
        _ptr(out16), dtype_code(out16_dtype) if out16 is not None else 2, _ptr(ws), nb, flags, _stream(stream)))
    return out if out16 is None else (out, out16)


def c2s(x, nbr, mask, mstart, gidx, m: int, cout: int, child_nbr, p: dict, plan=None, child_plan=None,
        cast_f32: bool = False, stream=None, out16_dtype=None, conv2_tiles=None):
    """The C2S block's features through tsp_c2s_ex, after its subdivision (mask uint8 [8N], mstart
    and gidx from subdivide, child_nbr the children's table): x f32 [N, Cin], p by reference
    names without the prefix ("norm1.weight", "norm1.bias", "conv1.weight" [8 Cout,27,Cin],
    "conv1.bias", "conv2.weight" [Cout,27,Cout], "conv2.bias"; optional "conv1.packed",
    "conv2.packed"). -> f32 [M, Cout], or (out, out rounded to out16_dtype) when out16_dtype is
    given. conv2_tiles, a list of (t0, nt) child-plan tile ranges: through tsp_c2s_part instead,
    the front part once, then conv2 over each range in turn."""
    torch = _torch()
    n, cin = x.shape
    if x.dtype != torch.float32:
        raise ValueError("x must be float32")
    _check_nbr(nbr, n, x.device)
    _check_nbr(child_nbr, m, x.device)
    if mask.dtype != torch.uint8 or mask.numel() != 8 * n:
        raise ValueError("mask must be uint8 with 8*N entries")
    if mstart.dtype != torch.int32 or mstart.numel() != n + 1 or gidx.dtype != torch.int32 or gidx.numel() < m:
        raise ValueError("mstart must be int32 [N+1] and gidx int32 [>= M]")
    t = {"conv1.weight": _mat(p["conv1.weight"], (8 * cout, 27, cin), "conv1.weight"),
         "conv2.weight": _mat(p["conv2.weight"], (cout, 27, cout), "conv2.weight")}
    for k, k_n in (("norm1.weight", cin), ("norm1.bias", cin), ("conv1.bias", 8 * cout), ("conv2.bias", cout)):
        t[k] = _vec(p[k], k_n, k)
    p1, p2 = p.get("conv1.packed"), p.get("conv2.packed")
    for pk, (ci_, co_), name in ((p1, (cin, 8 * cout), "conv1.packed"), (p2, (cout, cout), "conv2.packed")):
        if pk is not None and pk.numel() * pk.element_size() != lib().tsp_conv_weight_packed_bytes(ci_, co_):
            raise ValueError(f"{name} must hold the weight packed by conv_weight_pack")
    for pl, rows, name in ((plan, n, "plan"), (child_plan, m, "child_plan")):
        if pl is not None and (pl.dtype != torch.uint8 or pl.numel() < lib().tsp_conv_plan_bytes(rows)):
            raise ValueError(f"{name} must be a uint8 buffer of tsp_conv_plan_bytes")
    _require_cuda(x, nbr, mask, mstart, gidx, child_nbr, plan, child_plan, p1, p2, *t.values())
    w = C2SWeights(_ptr(t["norm1.weight"]), _ptr(t["norm1.bias"]), _ptr(t["conv1.weight"]),
                   dtype_code(t["conv1.weight"].dtype), _ptr(t["conv1.bias"]), _ptr(p1), _ptr(t["conv2.weight"]),
                   dtype_code(t["conv2.weight"].dtype), _ptr(t["conv2.bias"]), _ptr(p2))
    flags = BLOCK_CAST_F32 if cast_f32 else 0
    xc = x.contiguous()
    out = torch.empty((m, cout), dtype=torch.float32, device=x.device)
    out16 = None if out16_dtype is None else torch.empty((m, cout), dtype=out16_dtype, device=x.device)
    nb = lib().tsp_c2s_workspace_bytes(n, m, cin, cout, ctypes.byref(w), int(plan is not None),
                                       int(child_plan is not None), flags)
    ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=x.device)
    mk = mask.reshape(-1).contiguous()
    args = (_ptr(xc), n, cin, _ptr(nbr), _ptr(plan), _ptr(mk), _ptr(mstart), _ptr(gidx), m, cout, _ptr(child_nbr),
            _ptr(child_plan), ctypes.byref(w), _ptr(out), _ptr(out16), dtype_code(out16_dtype) if out16 is not None
            else 2, _ptr(ws), nb, flags)
    if conv2_tiles is None:
        _check("tsp_c2s_ex", lib().tsp_c2s_ex(*args, _stream(stream)))
    else:
        _check("tsp_c2s_part", lib().tsp_c2s_part(*args, 1, 0, -1, _stream(stream)))
        for t0, nt in conv2_tiles:
            _check("tsp_c2s_part", lib().tsp_c2s_part(*args, 2, t0, nt, _stream(stream)))
    return out if out16 is None else (out, out16)


# --------------------------------------------------------------------------------------------
# transformer pieces over packed rows
# --------------------------------------------------------------------------------------------
class _On:
    """Runs a call on its tensors' device and on the given stream: what it allocates there belongs to
    that stream, and its tensors are kept from reuse until the stream is past the call."""

    def __init__(self, device, stream, current):
        if stream is not None and stream.device != device:
            raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
        self.device, self.current, self.guards = device, current, []
        self.stream = stream if stream is not None else current

    def __enter__(self):
        torch = _torch()
        self.guards = [torch.cuda.device(self.device), torch.cuda.stream(self.stream)]
        for g in self.guards:
            g.__enter__()
        return self

    def __exit__(self, *exc):
        for g in reversed(self.guards):
            g.__exit__(*exc)

    def keep(self, *tensors):
        if self.stream != self.current:
            for t in tensors:
                if t is not None:
                    t.record_stream(self.stream)
                    t.record_stream(self.current)


def _nothing(*tensors):
    pass


def _current_stream(index: int) -> int:
    """The pointer of the device's current stream. torch's own call for it, which is not public, where there is
    one: a Stream object is 1 us, a tenth of the host's side of a call."""
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(index) if raw else torch.cuda.current_stream(index).cuda_stream


def _launch(device, stream, call, *args):
    """call(stream pointer, keep, *args) on the device and stream; keep(*tensors) is told every tensor the
    call uses."""
    torch = _torch()
    index = device.index
    if stream is None and index == torch.cuda.current_device():
        return call(_current_stream(index), _nothing, *args)
    with _On(device, stream, torch.cuda.current_stream(index)) as on:
        return call(on.stream.cuda_stream, on.keep, *args)


def _same_device(device, *named):
    """named: name, tensor, name, tensor, ..."""
    index = device.index      # (None: not a GPU's)
    if index is None or device.type != "cuda":
        raise ValueError("tensors must live on the GPU")
    for t in named[1::2]:
        if t is not None and t.get_device() != index:
            name = next(n for n, u in zip(named[::2], named[1::2]) if u is t)
            raise ValueError(f"{name} must live on {device}, got {t.device}")


def _p(t) -> int:
    return 0 if t is None else t.data_ptr()


def _offsets(t, name: str):
    """(offsets, samples) of packed rows; None: one sample."""
    if t is None:
        return None, 1
    if t.dtype != _torch().int32 or t.dim() != 1 or t.numel() < 2 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of samples + 1 entries")
    return t, t.numel() - 1


def _check_workspace(ws):
    # (its size is the library's to check)
    if ws.dtype != _torch().uint8 or not ws.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 buffer")


def group_norm_workspace(n: int, c: int, groups: int, samples: int = 1, device="cuda"):
    """The uint8 workspace group_norm needs for these sizes."""
    return _torch().empty(max(lib().tsp_group_norm_workspace_bytes(n, c, groups, samples), 16), dtype=_torch().uint8,
                          device=device)


def group_norm(x, groups: int, gamma=None, beta=None, eps: float = 1e-6, silu: bool = False, offsets=None, out_dtype=None,
               out=None, workspace=None, stream=None):
    """Group norm over packed samples, channels last: x [N, C], each sample's rows and a group's
    C / groups channels normalised together (biased variance) [* gamma + beta] [then SiLU]. offsets int32
    [samples + 1] on the GPU: the samples' first rows and the last one's end (None: one sample); rows
    outside every sample are left as they were in out. out [N, C] may be x (and must not overlap it otherwise); workspace
    (group_norm_workspace) may be given to reuse it."""
    torch = _torch()
    if x.dim() != 2 or groups < 1 or x.shape[1] % groups:
        raise ValueError(f"x must be [N, C] with C a multiple of groups={groups}, got {tuple(x.shape)}")
    n, c = x.shape
    dev = x.device
    offsets, samples = _offsets(offsets, "offsets")
    for name, t in (("gamma", gamma), ("beta", beta)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != c or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous float32 vector of {c}")
    if out is not None:
        _check_out(out, n, c, out_dtype or out.dtype, dev)
    _same_device(dev, "offsets", offsets, "gamma", gamma, "beta", beta, "workspace", workspace)
    xd = dtype_code(x.dtype)
    if workspace is not None:
        _check_workspace(workspace)

    def call(s, keep):
        xc = x.contiguous()
        o = out if out is not None else torch.empty((n, c), dtype=out_dtype or x.dtype, device=dev)
        ws = workspace
        if ws is None:
            ws = torch.empty(max(lib().tsp_group_norm_workspace_bytes(n, c, groups, samples), 16), dtype=torch.uint8, device=dev)
        g, b = _aligned(gamma), _aligned(beta)      # (the kernels would read all of x value by value otherwise)
        keep(x, xc, gamma, beta, g, b, offsets, o, ws)
        _check("tsp_group_norm",
               lib().tsp_group_norm(_p(xc), xd, n, c, groups, _p(offsets), samples, _p(g), _p(b), eps,
                                    1 if silu else 0, _p(o), dtype_code(o.dtype), _p(ws), ws.numel(), s))
        return o
    return _launch(dev, stream, call)


def _heads(t, n: int, h: int, d: int):
    """t [n, h, d] as tsp_heads, or None where the kernels cannot read it as it lies."""
    row, head, one = t.stride()
    p = t.data_ptr()
    if one == 1 and d <= row <= 1 << 20 and not (p & 15 or (row | head) & 7):
        return Heads(p, row, head)
    # (the stride of an axis of one may be anything)
    if p % 16 or (one != 1 and d != 1) or (n > 1 and (row % 8 or not d <= row <= 1 << 20)) or (h > 1 and head % 8):
        return None
    return Heads(p, row if n > 1 else h * d, head if h > 1 else d)


def _fitted(t, n: int, h: int, d: int):
    """(t [n, h, d], its tsp_heads), t copied where the kernels could not read it as it lies."""
    hd = _heads(t, n, h, d)
    if hd is None:
        t = t.clone(memory_format=_torch().contiguous_format)
        hd = _heads(t, n, h, d) or Heads(t.data_ptr(), h * d, d)   # (D not of whole pieces: the library refuses it)
    return t, hd


def _heads_out(out, n: int, h: int, d: int, dtype, device, name: str):
    """The tsp_heads of a caller's output."""
    if out.shape != (n, h, d) or out.dtype != dtype or out.device != device:
        raise ValueError(f"{name} must be {dtype} {[n, h, d]} on {device}")
    hd = _heads(out, n, h, d)
    if hd is None:
        raise ValueError(f"{name} must be 16-byte aligned with contiguous heads and strides that are multiples of 8")
    return hd


def _aligned(t):
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def rope_axes(q, pos, k=None, pairs=None, theta: float = 10000.0, interleaved: bool = True, q_gamma=None, k_gamma=None,
              eps: float = 1e-6, out_dtype=None, q_out=None, k_out=None, stream=None):
    """Rotary positions on several axes: q [N, Hq, D] (and k [N, Hk, D] in the same launch) turned by
    pos int32 [N, axes]. Pair j of axis a turns by pos[:, a] * theta ** (-j / pairs[a]); pairs defaults to
    D // 2 // axes on every axis, and a head's pairs after the last axis's stay as they are. Pairs are
    neighbours (2p, 2p + 1), or with interleaved=False (p, p + D/2). q_gamma [Hq, D] and k_gamma [Hk, D]
    (float32): every head is RMS-normalised first, x / sqrt(mean(x^2) + eps) * gamma. -> q's result, or the
    pair with k. Heads may be strided views; q_out and k_out may be q and k themselves."""
    torch = _torch()
    if q.dim() != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
        raise ValueError("q must be [N, Hq, D] and k [N, Hk, D]")
    n, hq, d = q.shape
    hk = 0 if k is None else k.shape[1]
    dev = q.device
    if k is not None and k.dtype != q.dtype:
        raise ValueError("q and k must have one dtype")
    if k is None and (k_gamma is not None or k_out is not None):
        raise ValueError("k_gamma and k_out need k")
    if pos.dtype != torch.int32 or pos.dim() != 2 or pos.shape[0] != n or not 1 <= pos.shape[1] <= 4:
        raise ValueError("pos must be int32 [N, axes] with 1 to 4 axes")
    axes = pos.shape[1]
    pairs = (d // 2 // axes,) * axes if pairs is None else tuple(map(int, pairs))
    if len(pairs) != axes:
        raise ValueError(f"pairs must name a count for each of {axes} axes")
    for name, g, h in (("q_gamma", q_gamma, hq), ("k_gamma", k_gamma, hk)):
        if g is not None and (g.dtype != torch.float32 or g.shape != (h, d) or not g.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous float32 {[h, d]}")
    _same_device(dev, "k", k, "pos", pos, "q_gamma", q_gamma, "k_gamma", k_gamma)
    odt = out_dtype or (q_out.dtype if q_out is not None else k_out.dtype if k_out is not None else q.dtype)
    qoh = None if q_out is None else _heads_out(q_out, n, hq, d, odt, dev, "q_out")
    koh = None if k_out is None else _heads_out(k_out, n, hk, d, odt, dev, "k_out")

    def call(s, keep):
        qc, qh = _fitted(q, n, hq, d)
        kc, kh = (None, None) if k is None else _fitted(k, n, hk, d)
        qo, ko, qoh_, koh_ = q_out, k_out, qoh, koh
        if qo is None:
            qo, qoh_ = _fitted(torch.empty((n, hq, d), dtype=odt, device=dev), n, hq, d)
        if k is not None and ko is None:
            ko, koh_ = _fitted(torch.empty((n, hk, d), dtype=odt, device=dev), n, hk, d)
        pc = pos.contiguous()
        gq, gk = _aligned(q_gamma), _aligned(k_gamma)
        keep(q, k, qc, kc, pos, pc, q_gamma, k_gamma, gq, gk, qo, ko)
        _check("tsp_rope_axes",
               lib().tsp_rope_axes(qh, hq, kh, hk, dtype_code(q.dtype), n, d, _p(pc), axes, (ctypes.c_int * axes)(*pairs), theta,
                                   0 if interleaved else 1, _p(gq), _p(gk), eps, qoh_, koh_, dtype_code(odt), s))
        return qo if k is None else (qo, ko)
    return _launch(dev, stream, call)


def attention_workspace(nq: int, nk: int, samples: int, hq: int, hkv: int, d: int, device="cuda"):
    """The uint8 workspace attention needs for these sizes."""
    return _torch().empty(max(lib().tsp_attention_workspace_bytes(nq, nk, samples, hq, hkv, d), 16), dtype=_torch().uint8,
                          device=device)


def attention(q, k, v, q_offsets=None, k_offsets=None, causal: bool = False, scale=None, out=None, workspace=None, stream=None):
    """Softmax attention within packed samples: q [Nq, Hq, D], k and v [Nk, Hkv, D] (one dtype, D a
    multiple of 8 up to 128, Hq a multiple of Hkv: head h of q reads head h // (Hq // Hkv)) -> [Nq, Hq, D].
    Row i of a sample sees all of the sample's keys, or with causal the keys j <= i + (Lk - Lq); a row that
    sees none gets zeros. q_offsets and k_offsets int32 [samples + 1] on the GPU: the samples' rows in q
    and in k and v (None, both: one sample); rows of out outside every sample are left as they were. scale
    defaults to D ** -0.5. 16-bit heads' probabilities are rounded to their type, float32 heads' are not (and take
    some ten times as long). Heads may be strided views; workspace (attention_workspace) may be given to
    reuse it."""
    torch = _torch()
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise ValueError("q must be [Nq, Hq, D], k and v [Nk, Hkv, D]")
    (nq, hq, d), (nk, hkv, _) = q.shape, k.shape
    dev = q.device
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have one dtype")
    if (q_offsets is None) != (k_offsets is None):
        raise ValueError("q_offsets and k_offsets come together")
    q_offsets, samples = _offsets(q_offsets, "q_offsets")
    k_offsets, k_samples = _offsets(k_offsets, "k_offsets")
    if samples != k_samples:
        raise ValueError("q_offsets and k_offsets must name the same samples")
    _same_device(dev, "k", k, "v", v, "q_offsets", q_offsets, "k_offsets", k_offsets, "workspace", workspace)
    given = None if out is None else _heads_out(out, nq, hq, d, q.dtype, dev, "out")
    if workspace is not None:
        _check_workspace(workspace)

    def call(s, keep):
        (qc, qh), (kc, kh), (vc, vh) = _fitted(q, nq, hq, d), _fitted(k, nk, hkv, d), _fitted(v, nk, hkv, d)
        o, oh = (out, given) if out is not None else _fitted(torch.empty((nq, hq, d), dtype=q.dtype, device=dev), nq, hq, d)
        ws = workspace
        if ws is None:
            need = lib().tsp_attention_workspace_bytes(nq, nk, samples, hq, hkv, d)
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        keep(q, k, v, qc, kc, vc, q_offsets, k_offsets, o, ws)
        _check("tsp_attention",
               lib().tsp_attention(qh, kh, vh, dtype_code(q.dtype), nq, nk, hq, hkv, d, _p(q_offsets), _p(k_offsets), samples,
                                   d ** -0.5 if scale is None else scale, 1 if causal else 0, oh, _p(ws),
                                   0 if ws is None else ws.numel(), s))
        return o
    return _launch(dev, stream, call)


# --------------------------------------------------------------------------------------------
# a served transformer block's step: RMS norm, linears on 8 bits, a paged cache and attention to it
# --------------------------------------------------------------------------------------------
class Mx(NamedTuple):
    """Rows in 8 bits: codes float8_e4m3fn [N, C], times a power of two for every 32 channels, float8_e8m0fnu
    [N, C / 32]."""
    codes: Any
    powers: Any


def mx_empty(n: int, c: int, device="cuda") -> Mx:
    """Buffers for [N, C] rows in 8 bits."""
    torch = _torch()
    if c % 32:
        raise ValueError(f"rows in 8 bits need a multiple of 32 channels, got {c}")
    return Mx(torch.empty((n, c), dtype=torch.float8_e4m3fn, device=device),
              torch.empty((n, c // 32), dtype=torch.float8_e8m0fnu, device=device))


def _check_mx(torch, m, n, c, name: str):
    """n and c may be None: any. -> (n, c)"""
    codes, powers = m
    shape, blocks = codes.shape, powers.shape
    if codes.dtype != torch.float8_e4m3fn or (powers.dtype != torch.float8_e8m0fnu and powers.dtype != torch.uint8) or len(shape) != 2:
        raise ValueError(f"{name} must be Mx(codes float8_e4m3fn [N, C], powers float8_e8m0fnu [N, C / 32])")
    rows, ch = shape
    if ch % 32 or blocks != (rows, ch // 32) or (n is not None and rows != n) or (c is not None and ch != c):
        raise ValueError(f"{name} has codes {list(shape)} and powers {list(blocks)}, expected {[n, c]} and one for 32 channels")
    if not (codes.is_contiguous() and powers.is_contiguous()):
        raise ValueError(f"{name} must be contiguous")
    return rows, ch


def rms_norm(x, gamma=None, eps: float = 1e-6, residual=None, residual_out=None, out_dtype=None, out=None, stream=None):
    """RMS norm of rows with the residual's addition: h = x [N, C] + residual, y = h / sqrt(mean(h^2) + eps) * gamma in
    fp32 -> y, or with a residual (y, h in the residual's dtype). out_dtype torch.float8_e4m3fn (or out an Mx): y in 8
    bits, as Mx, for linear_mx (C a multiple of 32). out and residual_out may be given; they may be x or residual where
    the dtypes agree."""
    torch = _torch()
    if x.dim() != 2:
        raise ValueError(f"x must be [N, C], got {tuple(x.shape)}")
    n, c = x.shape
    dev = x.device
    if gamma is not None and (gamma.dtype != torch.float32 or gamma.numel() != c or not gamma.is_contiguous()):
        raise ValueError(f"gamma must be a contiguous float32 vector of {c}")
    if residual is not None and tuple(residual.shape) != (n, c):
        raise ValueError(f"residual must be {[n, c]}, got {list(residual.shape)}")
    if residual_out is not None:
        if residual is None:
            raise ValueError("residual_out needs a residual")
        _check_out(residual_out, n, c, residual.dtype, dev)
    _same_device(dev, "gamma", gamma, "residual", residual)
    xd, rd = dtype_code(x.dtype), 0 if residual is None else dtype_code(residual.dtype)
    mx = isinstance(out, tuple) if out is not None else out_dtype == torch.float8_e4m3fn
    if mx:
        if out_dtype not in (None, torch.float8_e4m3fn):
            raise ValueError(f"out is in 8 bits, out_dtype {out_dtype}")
        if c % 32:
            raise ValueError(f"rows in 8 bits need a multiple of 32 channels, got {c}")
        if out is not None:
            _check_mx(torch, out, n, c, "out")
            _same_device(dev, "out", out[0], "out", out[1])
    elif out is not None:
        _check_out(out, n, c, out_dtype or out.dtype, dev)
    odt = None if mx else (out.dtype if out is not None else out_dtype or x.dtype)
    od = TSP_MX8 if mx else dtype_code(odt)

    def call(s, keep):
        xc, rc = x.contiguous(), None if residual is None else residual.contiguous()
        o = out
        if o is None:
            o = mx_empty(n, c, dev) if mx else torch.empty((n, c), dtype=odt, device=dev)
        codes, powers = o if mx else (o, None)
        ro = residual_out
        if ro is None and residual is not None:
            ro = torch.empty((n, c), dtype=residual.dtype, device=dev)
        g = _aligned(gamma)
        keep(x, xc, residual, rc, gamma, g, codes, powers, ro)
        _check("tsp_rms_norm", lib().tsp_rms_norm(_p(xc), xd, n, c, _p(rc), rd, _p(g), eps, _p(codes), od, _p(powers), _p(ro), s))
        return o if residual is None else (o, ro)
    return _launch(dev, stream, call)


def mx_quantize(x, out=None, stream=None) -> Mx:
    """x [N, C] rounded to 8 bits (C a multiple of 32): a layer's weight once, or rows that no norm precedes."""
    if x.dim() != 2 or x.shape[1] % 32:
        raise ValueError(f"x must be [N, C] with C a multiple of 32, got {tuple(x.shape)}")
    n, c = x.shape
    dev = x.device
    _same_device(dev)
    xd = dtype_code(x.dtype)
    if out is not None:
        _check_mx(_torch(), out, n, c, "out")
        _same_device(dev, "out", out[0], "out", out[1])

    def call(s, keep):
        xc = _aligned(x.contiguous())
        o = out if out is not None else mx_empty(n, c, dev)
        keep(x, xc, *o)
        _check("tsp_mx_quantize", lib().tsp_mx_quantize(_p(xc), xd, n, c, _p(o[0]), _p(o[1]), s))
        return o
    return _launch(dev, stream, call)


def linear_mx_workspace(n: int, ci: int, co: int, device="cuda"):
    """A workspace for linear_mx, which needs none: 16 bytes whatever the sizes."""
    return _torch().empty(max(lib().tsp_linear_mx_workspace_bytes(n, ci, co), 16), dtype=_torch().uint8, device=device)


def linear_mx(x, weight, bias=None, act: str = "none", residual=None, out_dtype=None, out=None, workspace=None, stream=None):
    """act(x W^T + bias) + residual on operands in 8 bits: x Mx of [N, Ci], weight Mx of [Co, Ci], bias float32 [Co],
    residual float32 [N, Co] -> [N, Co] in out_dtype (bfloat16 by default; float32 is added in fp32 throughout, at half
    the rate). out may be given, and be a float32 residual itself. workspace is taken as the other calls take theirs; none is
    needed."""
    torch = _torch()
    n, ci = _check_mx(torch, x, None, None, "x")
    co, _ = _check_mx(torch, weight, None, ci, "weight")
    (xc, xp), (wc, wp) = x, weight
    dev = xc.device
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != co or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous float32 vector of {co}")
    if residual is not None and (residual.dtype != torch.float32 or residual.shape != (n, co)):
        raise ValueError(f"residual must be float32 {[n, co]}")
    if out is not None:
        _check_out(out, n, co, out_dtype or out.dtype, dev)
    _same_device(dev, "x's powers", xp, "weight's codes", wc, "weight's powers", wp, "bias", bias, "residual", residual, "workspace", workspace)
    if workspace is not None:
        _check_workspace(workspace)
    odt = out.dtype if out is not None else out_dtype or torch.bfloat16
    od, ac = dtype_code(odt), ACT[act]

    def call(s, keep):
        rc = None if residual is None else residual.contiguous()
        o = out if out is not None else torch.empty((n, co), dtype=odt, device=dev)
        xa, pa, wa, qa = _aligned(xc), _aligned(xp), _aligned(wc), _aligned(wp)
        keep(xc, xp, wc, wp, xa, pa, wa, qa, bias, residual, rc, o, workspace)
        _check("tsp_linear_mx",
               lib().tsp_linear_mx(xa.data_ptr(), pa.data_ptr(), n, ci, wa.data_ptr(), qa.data_ptr(), _p(bias), co, ac, _p(rc),
                                   o.data_ptr(), od, _p(workspace), 0 if workspace is None else workspace.numel(), s))
        return o
    return _launch(dev, stream, call)


class KVCache:
    """A paged cache of keys and values: data uint8 [pages, bytes of a page], each page of `page` tokens (16, 32, 64, 128 or
    256) of `heads` heads of d elements (a multiple of 8 up to 128), held as `dtype`: "mx4" (4 bits with a power of two for
    every 32 elements), torch.float16 or torch.bfloat16. Made by kv_cache."""

    def __init__(self, data, page: int, heads: int, d: int, dtype):
        torch = _torch()
        self.format = TSP_KV_MX4 if dtype == "mx4" else dtype_code(dtype) if dtype in (torch.float16, torch.bfloat16) else None
        if self.format is None:
            raise ValueError(f'a cache holds "mx4", float16 or bfloat16, not {dtype}')
        size = lib().tsp_kv_page_bytes(page, heads, d, self.format)
        if not size:
            raise ValueError(f"no cache of pages of {page} tokens (16, 32, 64, 128 or 256), {heads} heads of {d} (a multiple of 8 up to 128)")
        if data.dtype != torch.uint8 or data.dim() != 2 or data.shape[1] != size or not data.is_contiguous() or data.data_ptr() % 16:
            raise ValueError(f"data must be a contiguous uint8 [pages, {size}], 16-byte aligned")
        self._data, self.page, self.heads, self.d, self.dtype = data, page, heads, d, dtype
        self.pages = data.shape[0]
        self.arg = KvCacheArg(data.data_ptr(), self.pages, page, heads, d, self.format)

    @property
    def data(self):
        """The pages (one tensor for the cache's life: calls hold its address)."""
        return self._data


def kv_cache(pages: int, page: int, heads: int, d: int, dtype="mx4", device="cuda") -> KVCache:
    """A cache of that many pages, all zeros."""
    torch = _torch()
    code = TSP_KV_MX4 if dtype == "mx4" else dtype_code(dtype) if dtype in (torch.float16, torch.bfloat16) else -1
    size = lib().tsp_kv_page_bytes(page, heads, d, code)
    return KVCache(torch.zeros((pages, size), dtype=torch.uint8, device=device), page, heads, d, dtype)


def _cache_places(cache, table, lengths, offsets, dev, *named):
    """Checks of a cache's table, lengths and rows' offsets, and of the device of theirs and the tensors named
    -> (offsets, samples, the table's columns)."""
    int32 = _torch().int32
    offsets, samples = _offsets(offsets, "offsets")
    shape = table.shape
    if table.dtype != int32 or len(shape) != 2 or shape[0] != samples or not shape[1] or not table.is_contiguous():
        raise ValueError(f"table must be a contiguous int32 [{samples}, max_pages]")
    if lengths.dtype != int32 or lengths.shape != (samples,) or not lengths.is_contiguous():
        raise ValueError(f"lengths must be a contiguous int32 [{samples}]")
    _same_device(dev, "cache", cache._data, "table", table, "lengths", lengths, "offsets", offsets, *named)
    return offsets, samples, shape[1]


def kv_append(cache: KVCache, k, v, table, lengths, offsets=None, q=None, pos=None, pairs=None, theta: float = 10000.0,
              interleaved: bool = True, q_gamma=None, k_gamma=None, eps: float = 1e-6, q_out=None, stream=None):
    """New keys and values k, v [N, Hkv, D] of packed samples into the cache, turned to their positions on the way. Of sample
    s with m rows (offsets int32 [samples + 1]; None: one sample), row i becomes key lengths[s] - m + i (lengths int32
    [samples]: the samples' keys after the call, counted from as they are), in page table[s, key // page] of the int32 table
    [samples, max_pages].
    pos int32 [N, axes], pairs, theta, interleaved and the gammas are rope_axes'; pos None: no turning. q [N, Hq, D] is
    normalised and turned in the same launch -> q's result (None without q); rows that are no sample's are left as
    they were in q_out, and in none. Keys whose place is not one of the cache's are not written; two rows must not have
    one place. q_out may be q itself."""
    torch = _torch()
    if k.dim() != 3 or v.shape != k.shape or k.shape[1:] != (cache.heads, cache.d):
        raise ValueError(f"k and v must be [N, {cache.heads}, {cache.d}]")
    n, hkv, d = k.shape
    dev = k.device
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError("q, k and v must have one dtype")
    if q is None and (q_gamma is not None or q_out is not None):
        raise ValueError("q_gamma and q_out need q")
    if q is not None and (q.dim() != 3 or q.shape[0] != n or q.shape[2] != d):
        raise ValueError(f"q must be [{n}, Hq, {d}]")
    hq = 0 if q is None else q.shape[1]
    offsets, samples, columns = _cache_places(cache, table, lengths, offsets, dev, "q", q, "v", v, "pos", pos, "q_gamma", q_gamma,
                                              "k_gamma", k_gamma)
    axes = 0
    if pos is not None:
        if pos.dtype != torch.int32 or pos.dim() != 2 or pos.shape[0] != n or not 1 <= pos.shape[1] <= 4:
            raise ValueError("pos must be int32 [N, axes] with 1 to 4 axes")
        axes = pos.shape[1]
        pairs = (d // 2 // axes,) * axes if pairs is None else tuple(map(int, pairs))
        if len(pairs) != axes:
            raise ValueError(f"pairs must name a count for each of {axes} axes")
    for name, g, h in (("q_gamma", q_gamma, hq), ("k_gamma", k_gamma, hkv)):
        if g is not None and (g.dtype != torch.float32 or g.shape != (h, d) or not g.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous float32 {[h, d]}")
    given = None if q_out is None else _heads_out(q_out, n, hq, d, k.dtype, dev, "q_out")
    code = dtype_code(k.dtype)

    def call(s, keep):
        (kc, kh), (vc, vh) = _fitted(k, n, hkv, d), _fitted(v, n, hkv, d)
        qc = qh = qo = qoh = None
        if q is not None:
            qc, qh = _fitted(q, n, hq, d)
            qo, qoh = (q_out, given) if q_out is not None else _fitted(torch.empty((n, hq, d), dtype=q.dtype, device=dev), n, hq, d)
        pc = None if pos is None else pos.contiguous()
        gq, gk = _aligned(q_gamma), _aligned(k_gamma)
        keep(k, v, q, kc, vc, qc, qo, pos, pc, q_gamma, k_gamma, gq, gk, table, lengths, offsets, cache._data)
        _check("tsp_kv_append",
               lib().tsp_kv_append(cache.arg, kh, vh, code, n, _p(offsets), samples, _p(table), columns, _p(lengths), qh, hq,
                                   _p(pc), axes, (ctypes.c_int * axes)(*pairs) if axes else None, theta, 0 if interleaved else 1,
                                   _p(gq), _p(gk), eps, qoh, s))
        return qo
    return _launch(dev, stream, call)


def kv_gather(cache: KVCache, table, lengths, offsets=None, n=None, out_dtype=None, k_out=None, v_out=None, stream=None):
    """Keys and values out of the cache -> packed (k, v) [N, Hkv, D] in out_dtype (bfloat16 by default, a 16-bit cache's own):
    of sample s with m rows (offsets; None: one sample of n), row i is key lengths[s] - m + i, zeros where the cache does
    not hold it; rows that are no sample's are left as they were. N is k_out's and v_out's, or n."""
    torch = _torch()
    dev = cache.data.device
    for name, o in (("k_out", k_out), ("v_out", v_out)):
        if o is not None and o.dim() == 3 and n is None:
            n = o.shape[0]
    if n is None:
        raise ValueError("the number of rows: k_out, v_out or n")
    offsets, samples, columns = _cache_places(cache, table, lengths, offsets, dev)
    odt = out_dtype or (k_out.dtype if k_out is not None else v_out.dtype if v_out is not None
                        else torch.bfloat16 if cache.dtype == "mx4" else cache.dtype)
    h, d = cache.heads, cache.d
    kg = None if k_out is None else _heads_out(k_out, n, h, d, odt, dev, "k_out")
    vg = None if v_out is None else _heads_out(v_out, n, h, d, odt, dev, "v_out")
    code = dtype_code(odt)

    def call(s, keep):
        ko, kh = (k_out, kg) if k_out is not None else _fitted(torch.empty((n, h, d), dtype=odt, device=dev), n, h, d)
        vo, vh = (v_out, vg) if v_out is not None else _fitted(torch.empty((n, h, d), dtype=odt, device=dev), n, h, d)
        keep(ko, vo, table, lengths, offsets, cache._data)
        _check("tsp_kv_gather", lib().tsp_kv_gather(cache.arg, n, _p(offsets), samples, _p(table), columns, _p(lengths), kh, vh, code, s))
        return ko, vo
    return _launch(dev, stream, call)


def attention_cached_workspace(nq: int, samples: int, hq: int, cache: KVCache, max_pages: int):
    """The uint8 workspace attention_cached needs for these sizes."""
    return _torch().empty(max(lib().tsp_attention_cached_workspace_bytes(nq, samples, hq, cache.arg, max_pages), 16),
                          dtype=_torch().uint8, device=cache.data.device)


def attention_cached(q, cache: KVCache, table, lengths, offsets=None, causal: bool = True, scale=None, out=None, workspace=None,
                     stream=None):
    """Softmax attention of q [Nq, Hq, D] (float16 or bfloat16; a 16-bit cache's dtype) to its samples' cached keys ->
    [Nq, Hq, D]. Of sample s with m rows (offsets int32 [samples + 1]; None: one sample), row i sees all lengths[s] keys, or
    with causal those with j <= i + (lengths[s] - m): after kv_append with the same lengths, its own key and those before. A
    row that sees none gets zeros; rows of out outside every sample are left as they were. Lengths are cut to what the table
    reaches. Hq is a multiple of the cache's heads, scale defaults to D ** -0.5; workspace (attention_cached_workspace) may be
    given to reuse it. A prompt beside many single tokens is better a call of its own."""
    torch = _torch()
    if q.dim() != 3 or q.shape[2] != cache.d or q.shape[1] % cache.heads:
        raise ValueError(f"q must be [Nq, Hq, {cache.d}] with Hq a multiple of {cache.heads}, got {list(q.shape)}")
    nq, hq, d = q.shape
    dev = q.device
    if q.dtype not in (torch.float16, torch.bfloat16) or (cache.dtype != "mx4" and cache.dtype != q.dtype):
        raise ValueError(f"q must be float16 or bfloat16, and a 16-bit cache's dtype; got {q.dtype} on {cache.dtype}")
    offsets, samples, columns = _cache_places(cache, table, lengths, offsets, dev, "workspace", workspace)
    given = None if out is None else _heads_out(out, nq, hq, d, q.dtype, dev, "out")
    if workspace is not None:
        _check_workspace(workspace)
    code = dtype_code(q.dtype)

    def call(s, keep):
        qc, qh = _fitted(q, nq, hq, d)
        o, oh = (out, given) if out is not None else _fitted(torch.empty((nq, hq, d), dtype=q.dtype, device=dev), nq, hq, d)
        ws = workspace
        if ws is None:
            need = lib().tsp_attention_cached_workspace_bytes(nq, samples, hq, cache.arg, columns)
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        keep(q, qc, o, ws, table, lengths, offsets, cache._data)
        _check("tsp_attention_cached",
               lib().tsp_attention_cached(qh, code, nq, hq, cache.arg, _p(offsets), samples, _p(table), columns, _p(lengths),
                                          d ** -0.5 if scale is None else scale, 1 if causal else 0, oh, _p(ws), ws.numel(), s))
        return o
    return _launch(dev, stream, call)
