"""ctypes binding of ``libsparseconv_b200.so`` (the C ABI declared in
``include/sparseconv_b200.h``) plus the tensor-level helpers the front end calls.

There is no CPU fallback: if the library is missing, or a tensor is not on a CUDA device,
every call raises. Outputs are allocated from torch's caching allocator and every launch
goes to ``torch.cuda.current_stream()``.

Device-side problems (coordinates out of range, a full table, a kernel wait limit) are
OR-ed into a per-device int32 status word. After each op the word is copied
asynchronously to pinned host memory; the next op on that device (or an explicit
``check_errors()``) raises ``RuntimeError`` if a bit is set. The linear and norm ops, which are
also called on a few rows, where a copy and an event would cost more than the op, give their
kernels a word in pinned host memory instead: a kernel writes there only on a problem, and the
next op on the device that checks (clipping, whose kernels report nothing, among them) reads it without
any call to CUDA. With the environment variable ``SPARSECONV_SYNC_CHECK=1`` each op synchronises and
checks at once; the linear, norm and clipping ops read the variable when this module is imported.
"""
from __future__ import annotations

import array
import ctypes
import functools
import operator
import os
import threading
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libsparseconv_b200.so")

SPCONV_OK, SPCONV_ERR_ARG, SPCONV_ERR_CUDA, SPCONV_ERR_UNSUPPORTED = 0, 1, 2, 3
STATUS_COORD_RANGE, STATUS_TABLE_FULL, STATUS_DUPLICATE, STATUS_WAIT_TIMEOUT = 1, 2, 4, 8
STATUS_OFFSETS = 16
DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
KERNEL_AUTO, KERNEL_SIMT, KERNEL_TCGEN05 = 0, 1, 2
NOALLOC_MAX_COORDS = 262144   # SPCONV_NOALLOC_MAX_COORDS
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}   # SPCONV_ACT_*
NORMS = {"none": 0, "layer": 1, "rms": 2}                    # SPCONV_NORM_*
CLIP_P2, CLIP_INF = 0, 1

_c_i64, _c_int, _c_void_p = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p



class ChannelParam(ctypes.Structure):
    """spconv_channel_param"""
    _fields_ = [("data", _c_void_p), ("grad", _c_void_p), ("dtype", _c_int), ("per_sample", _c_int)]


class ResidualNormArgs(ctypes.Structure):
    """spconv_residual_norm_args"""
    _fields_ = [("dtype", _c_int), ("channels", _c_int), ("num_rows", _c_i64),
                ("feats", _c_void_p), ("residual", _c_void_p), ("hidden", _c_void_p), ("normed", _c_void_p),
                ("grad_hidden", _c_void_p), ("grad_normed", _c_void_p),
                ("grad_feats", _c_void_p), ("grad_residual", _c_void_p), ("row_stats", _c_void_p),
                ("gate", ChannelParam), ("weight", ChannelParam), ("bias", ChannelParam),
                ("next_weight", ChannelParam), ("next_bias", ChannelParam),
                ("offsets", _c_void_p), ("num_samples", _c_int), ("norm", _c_int), ("next_norm", _c_int),
                ("residual_scale", ctypes.c_float), ("eps", ctypes.c_float),
                ("workspace", _c_void_p), ("workspace_bytes", _c_i64), ("status", _c_void_p)]


# name -> (restype, argtypes); the order mirrors include/sparseconv_b200.h
SIGNATURES = {
    "spconv_abi_version": (_c_int, []),
    "spconv_last_error": (ctypes.c_char_p, []),
    "spconv_hashmap_capacity": (_c_i64, [_c_i64]),
    "spconv_mask_words": (_c_int, [_c_int]),
    "spconv_neighbor_map_workspace_bytes": (_c_i64, [_c_i64, _c_int, _c_int, _c_int, _c_int]),
    "spconv_build_submanifold_neighbor_map": (_c_int, [
        _c_void_p, _c_i64, _c_int, _c_int, _c_int, _c_int,
        _c_int, _c_int, _c_int, _c_int, _c_int, _c_int,
        _c_void_p, _c_i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "spconv_submanifold_conv_forward": (_c_int, [
        _c_void_p, _c_int, _c_i64, _c_int, _c_void_p, _c_void_p, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "spconv_submanifold_conv_forward_ex": (_c_int, [
        _c_void_p, _c_int, _c_i64, _c_int, _c_void_p, _c_void_p, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int]),
    "spconv_conv_splitk_workspace_bytes": (_c_i64, [_c_i64, _c_int]),
    "spconv_submanifold_conv_forward_splitk": (_c_int, [
        _c_void_p, _c_int, _c_i64, _c_int, _c_void_p, _c_void_p, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_i64, _c_void_p, _c_void_p, _c_void_p]),
    "spconv_build_submanifold_neighbor_map_noalloc": (_c_int, [
        _c_void_p, _c_i64, _c_int, _c_int, _c_int, _c_int,
        _c_int, _c_int, _c_int, _c_int, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "spconv_neighbor_map_2d_workspace_bytes": (_c_i64, [_c_i64, _c_int, _c_int, _c_int]),
    "spconv_build_submanifold_neighbor_map_2d": (_c_int, [
        _c_void_p, _c_i64, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int,
        _c_void_p, _c_i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "spconv_from_dense_workspace_bytes": (_c_i64, [_c_int, _c_int, _c_int, _c_int]),
    "spconv_from_dense": (_c_int, [
        _c_void_p, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _c_void_p, _c_i64, _c_void_p,
        _c_void_p, _c_void_p, _c_i64, _c_int, _c_void_p]),
    "spconv_to_dense": (_c_int, [
        _c_void_p, _c_int, _c_void_p, _c_i64, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_void_p]),
    "spconv_hashmap_insert": (_c_int, [
        _c_void_p, _c_void_p, _c_i64, _c_int, _c_int, _c_void_p, _c_void_p, _c_i64, _c_void_p, _c_void_p]),
    "spconv_hashmap_lookup": (_c_int, [
        _c_void_p, _c_void_p, _c_i64, _c_int, _c_int, _c_void_p, _c_void_p, _c_i64, _c_void_p]),
    "spconv_submanifold_conv_backward_input": (_c_int, [
        _c_void_p, _c_int, _c_i64, _c_int, _c_void_p, _c_int, _c_int, _c_void_p, _c_void_p, _c_void_p,
        _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "spconv_transpose_neighbor_map": (_c_int, [
        _c_void_p, _c_i64, _c_int, _c_void_p, _c_void_p, _c_void_p, _c_void_p]),
    "spconv_weight_grad_workspace_bytes": (_c_i64, [_c_i64, _c_int]),
    "spconv_submanifold_conv_weight_grad": (_c_int, [
        _c_void_p, _c_void_p, _c_int, _c_i64, _c_int, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_i64, _c_void_p, _c_void_p]),
    "spconv_linear_forward_workspace_bytes": (_c_i64, [_c_int, _c_i64, _c_int, _c_int, _c_int, _c_int]),
    "spconv_linear_forward": (_c_int, [
        _c_void_p, _c_int, _c_i64, _c_int, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_void_p, _c_i64, _c_int, _c_void_p, _c_void_p]),
    "spconv_linear_forward_ex": (_c_int, [
        _c_void_p, _c_int, _c_i64, _c_int, _c_void_p, _c_void_p, _c_int, _c_void_p, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_void_p, _c_i64, _c_int, _c_void_p, _c_void_p]),
    "spconv_linear_backward_workspace_bytes": (_c_i64, [_c_int, _c_i64, _c_int, _c_int, _c_int]),
    "spconv_linear_backward": (_c_int, [
        _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_i64, _c_int, _c_int, _c_int,
        _c_void_p, _c_void_p, _c_int, _c_void_p, _c_int, _c_void_p, _c_i64, _c_int, _c_void_p, _c_void_p]),
    "spconv_residual_norm_workspace_bytes": (_c_i64, [_c_i64, _c_int, _c_int]),
    "spconv_residual_norm_forward": (_c_int, [ctypes.POINTER(ResidualNormArgs), _c_void_p]),
    "spconv_residual_norm_backward": (_c_int, [ctypes.POINTER(ResidualNormArgs), _c_void_p]),
    "spconv_clip_gradients_workspace_bytes": (_c_i64, [_c_int]),
    "spconv_clip_gradients": (_c_int, [
        _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_int, ctypes.c_float, _c_void_p,
        _c_void_p, _c_i64, _c_void_p]),
    "spconv_set_wait_limit_ns": (ctypes.c_uint64, [ctypes.c_uint64]),
    "spconv_stage_timing": (_c_int, [_c_int]),
    "spconv_stage_times_ms": (_c_int, [_c_void_p, _c_void_p, _c_int]),
}

STAGES = ("memset", "insert", "map", "order", "conv")

_lib = None
_lock = threading.Lock()


def load_library(path: Optional[str] = None) -> ctypes.CDLL:
    """Load the CUDA library (once). Raises RuntimeError if it has not been built."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = path or LIB_PATH
    if not os.path.exists(p):
        raise RuntimeError(
            f"sparseconv CUDA library not found at {p}; build it with "
            "`python sparse-conv_b200/build.py` (there is no CPU fallback)")
    lib = ctypes.CDLL(p)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if lib.spconv_abi_version() != 1:
        raise RuntimeError("sparseconv CUDA library ABI version mismatch")
    if path is None:
        _lib = lib
    return lib


def _raise(rc: int, what: str) -> None:
    msg = load_library().spconv_last_error().decode(errors="replace")
    if rc == SPCONV_ERR_ARG:
        raise ValueError(f"{what}: {msg}")
    if rc == SPCONV_ERR_UNSUPPORTED:
        raise NotImplementedError(f"{what}: {msg}")
    raise RuntimeError(f"{what}: {msg}")


def _stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(*tensors: torch.Tensor) -> torch.device:
    first = tensors[0]
    if first.is_cuda:
        index = first.get_device()
        for t in tensors:
            if t is not None and t.get_device() != index:      # -1 on the CPU
                break
        else:
            return first.device
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(
                "sparseconv runs on CUDA devices only (no CPU fallback); got a tensor on "
                f"{t.device}")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    return dev


def refuse_forward_mode(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Raises for a tensor with a forward-mode tangent. A call that needs no gradients does not pass
    through autograd, which would raise, and its result would count as constant."""
    if getattr(forward_ad, "_current_level", 0) < 0:         # outside of every dual_level: one comparison
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative")


# ---------------------------------------------------------------------------------------
# Device status word and deferred checks.
# ---------------------------------------------------------------------------------------
class _DeviceStatus:
    def __init__(self, device: torch.device):
        self.device = device
        self.word = torch.zeros(1, dtype=torch.int32, device=device)
        self.host = torch.zeros(1, dtype=torch.int32, pin_memory=True)
        self.event = torch.cuda.Event()
        self.pending = False
        # written by kernels that have a problem, read here directly (mapped pinned memory)
        self.mapped = torch.zeros(1, dtype=torch.int32, pin_memory=True)
        self.mapped_ptr = self.mapped.data_ptr()
        self.mapped_word = ctypes.c_int32.from_address(self.mapped_ptr)


_status = {}


def status_word(device: torch.device) -> _DeviceStatus:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    st = _status.get(idx)
    if st is None:
        with _lock:
            st = _status.get(idx)
            if st is None:
                st = _DeviceStatus(torch.device("cuda", idx))
                _status[idx] = st
    return st


def describe_status(bits: int) -> str:
    parts = []
    if bits & STATUS_COORD_RANGE:
        parts.append("a coordinate lies outside the spatial shape [0,N)x[0,W)x[0,H)x[0,D)")
    if bits & STATUS_TABLE_FULL:
        parts.append("the coordinate hash table overflowed")
    if bits & STATUS_WAIT_TIMEOUT:
        parts.append("a kernel-internal wait reached its time limit")
    if bits & STATUS_OFFSETS:
        parts.append("sample offsets do not ascend from 0 to the number of rows")
    return "; ".join(parts)


_FATAL_BITS = STATUS_COORD_RANGE | STATUS_TABLE_FULL | STATUS_WAIT_TIMEOUT | STATUS_OFFSETS


def _inspect(st: _DeviceStatus) -> None:
    bits = int(st.host.item())
    st.pending = False
    if bits & _FATAL_BITS:
        st.word.zero_()
        raise RuntimeError(f"sparseconv device error: {describe_status(bits)} (status bits {bits:#x})")


def after_launch(device: torch.device) -> None:
    """Queue the status read-back of this op; check at once if SPARSECONV_SYNC_CHECK=1.

    Skipped while the stream is being captured into a CUDA graph (call ``check_errors``
    after replays instead)."""
    if torch.cuda.is_current_stream_capturing():
        return
    st = status_word(device)
    stream = torch.cuda.current_stream(device)
    st.host.copy_(st.word, non_blocking=True)
    st.event.record(stream)
    st.pending = True
    if os.environ.get("SPARSECONV_SYNC_CHECK", "0") == "1":
        st.event.synchronize()
        _inspect(st)


def before_launch(device: torch.device) -> None:
    """Raise for an error found by an earlier op on this device, if its read-back landed or it is in
    the host's word."""
    if torch.cuda.is_current_stream_capturing():
        return
    st = status_word(device)
    if st.mapped_word.value:
        _inspect_mapped(st)
    if st.pending and st.event.query():
        _inspect(st)


def _inspect_mapped(st: _DeviceStatus) -> None:
    bits = st.mapped_word.value
    if bits:
        st.mapped_word.value = 0
        if bits & _FATAL_BITS:
            raise RuntimeError(f"sparseconv device error: {describe_status(bits)} (status bits {bits:#x})")


def mapped_status(index: int) -> int:
    """Address of the device's host status word, for an op about to launch; raises for an error
    that an earlier op reported there."""
    st = _status.get(index) or status_word(torch.device("cuda", index))
    if st.mapped_word.value:
        _inspect_mapped(st)
    return st.mapped_ptr


# read once, for the ops whose host time counts
_SYNC_CHECK = os.environ.get("SPARSECONV_SYNC_CHECK", "0") == "1"


def after_mapped_launch(index: int) -> None:
    """Check at once if SPARSECONV_SYNC_CHECK=1 at import (not while the stream is being captured)."""
    if _SYNC_CHECK and not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(index).synchronize()
        _inspect_mapped(_status[index])


def check_errors(device: Optional[torch.device] = None) -> int:
    """Synchronise with the device's status read-back and raise on an error.

    Returns the status bits seen (duplicate coordinates are reported, not raised).
    """
    devs = [status_word(device)] if device is not None else list(_status.values())
    bits = 0
    for st in devs:
        if st.pending:
            st.event.synchronize()
        torch.cuda.synchronize(st.device)
        st.host.copy_(st.word)
        bits |= int(st.host.item()) | st.mapped_word.value
        _inspect(st)
        _inspect_mapped(st)
    return bits


def reset_status(device: Optional[torch.device] = None) -> None:
    for st in ([status_word(device)] if device is not None else list(_status.values())):
        st.word.zero_()
        st.pending = False
        st.mapped_word.value = 0


# ---------------------------------------------------------------------------------------
# Tensor-level calls.
# ---------------------------------------------------------------------------------------
def mask_words(kernel_volume: int) -> int:
    return int(load_library().spconv_mask_words(int(kernel_volume)))


def hashmap_capacity(num_coords: int) -> int:
    return int(load_library().spconv_hashmap_capacity(int(num_coords)))


def workspace_bytes(num_coords: int, batch: int, W: int, H: int, D: int) -> int:
    return int(load_library().spconv_neighbor_map_workspace_bytes(int(num_coords), batch, W, H, D))


def build_neighbor_map(coords: torch.Tensor, batch: int, W: int, H: int, D: int,
                       kernel_size: Sequence[int], dilation: Sequence[int],
                       workspace: Optional[torch.Tensor] = None,
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Kernel map of ``coords`` ([M,4] int32 on CUDA): (neighbor_map [M,V] int32,
    masks [M,ceil(V/32)] int32 bit patterns, order [M] int32)."""
    lib = load_library()
    dev = _require_cuda(coords)
    if coords.dtype != torch.int32 or coords.dim() != 2 or coords.shape[1] != 4:
        raise ValueError("coords must be an [M, 4] int32 tensor")
    if not coords.is_contiguous():
        raise ValueError("coords must be contiguous")
    Kw, Kh, Kd = (int(k) for k in kernel_size)
    Dw, Dh, Dd = (int(d) for d in dilation)
    M = int(coords.shape[0])
    V = Kw * Kh * Kd
    MW = max(1, mask_words(V))
    nbr = torch.empty((M, V), dtype=torch.int32, device=dev)
    masks = torch.empty((M, MW), dtype=torch.int32, device=dev)
    order = torch.empty((M,), dtype=torch.int32, device=dev)
    if M == 0:
        return nbr, masks, order
    need = workspace_bytes(M, batch, W, H, D)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty((need,), dtype=torch.uint8, device=dev)
    before_launch(dev)
    st = status_word(dev)
    rc = lib.spconv_build_submanifold_neighbor_map(
        coords.data_ptr(), M, int(batch), int(W), int(H), int(D), Kw, Kh, Kd, Dw, Dh, Dd,
        workspace.data_ptr(), need, nbr.data_ptr(), masks.data_ptr(), order.data_ptr(),
        st.word.data_ptr(), _stream_ptr(dev))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_build_submanifold_neighbor_map")
    return nbr, masks, order


def build_neighbor_map_2d(coords: torch.Tensor, batch: int, W: int, H: int,
                          kernel_size: Sequence[int], dilation: Sequence[int],
                          ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """2-D kernel map of ``coords`` ([M,3] int32 (b, x, y) on CUDA): (neighbor_map [M, Kw*Kh]
    int32, masks, order), the map of the reference's
    ``hashmap_build_submanifold_conv2d_neighbor_map_cuda_naive`` (neighbor_map.cu:10-111)."""
    lib = load_library()
    dev = _require_cuda(coords)
    if coords.dtype != torch.int32 or coords.dim() != 2 or coords.shape[1] != 3:
        raise ValueError("coords must be an [M, 3] int32 tensor")
    if not coords.is_contiguous():
        raise ValueError("coords must be contiguous")
    Kw, Kh = (int(k) for k in kernel_size)
    Dw, Dh = (int(d) for d in dilation)
    M = int(coords.shape[0])
    V = Kw * Kh
    nbr = torch.empty((M, V), dtype=torch.int32, device=dev)
    masks = torch.empty((M, max(1, mask_words(V))), dtype=torch.int32, device=dev)
    order = torch.empty((M,), dtype=torch.int32, device=dev)
    if M == 0:
        return nbr, masks, order
    need = int(lib.spconv_neighbor_map_2d_workspace_bytes(M, int(batch), int(W), int(H)))
    if need < 0:
        raise ValueError("invalid 2-D map arguments")
    workspace = torch.empty((need,), dtype=torch.uint8, device=dev)
    before_launch(dev)
    st = status_word(dev)
    rc = lib.spconv_build_submanifold_neighbor_map_2d(
        coords.data_ptr(), M, int(batch), int(W), int(H), Kw, Kh, Dw, Dh, workspace.data_ptr(), need,
        nbr.data_ptr(), masks.data_ptr(), order.data_ptr(), st.word.data_ptr(), _stream_ptr(dev))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_build_submanifold_neighbor_map_2d")
    return nbr, masks, order


def conv_forward(feats: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                 nbr: torch.Tensor, masks: Optional[torch.Tensor], order: Optional[torch.Tensor],
                 kernel: int = KERNEL_AUTO, out: Optional[torch.Tensor] = None,
                 split: bool = False) -> torch.Tensor:
    """out[i] = bias + sum_v feats[nbr[i,v]] @ weight[:, v, :]^T over valid neighbours.

    ``weight`` is [Co, V, Ci] (or [Co, Kw, Kh, Kd, Ci]) in the dtype of ``feats``. ``split``
    runs the split-K variant (``spconv_submanifold_conv_forward_splitk``: the heaviest tiles'
    offsets spread over two CTAs, fp32 partials in a workspace from torch's allocator).
    """
    lib = load_library()
    dev = _require_cuda(feats, weight, bias, nbr, masks, order)
    if feats.dtype not in DTYPE_CODES:
        raise TypeError(f"unsupported feature dtype {feats.dtype}")
    if not feats.is_contiguous():
        raise ValueError("feats must be contiguous")
    M, Ci = int(feats.shape[0]), int(feats.shape[1])
    Co = int(weight.shape[0])
    V = int(nbr.shape[1]) if nbr.dim() == 2 else 0
    if nbr.shape[0] != M:
        raise ValueError(f"neighbor map has {nbr.shape[0]} rows for {M} feature rows")
    w = weight.reshape(Co, V, Ci)
    if w.dtype != feats.dtype:
        w = w.to(feats.dtype)
    w = w.contiguous()
    b = None
    if bias is not None:
        b = bias.to(feats.dtype).contiguous()
        if b.numel() != Co:
            raise ValueError(f"bias has {b.numel()} entries for {Co} output channels")
    nb = nbr.view(torch.int32) if nbr.dtype == torch.uint32 else nbr
    if nb.dtype != torch.int32 or not nb.is_contiguous():
        raise ValueError("neighbor map must be a contiguous [M, V] int32/uint32 tensor")
    mk = None
    if masks is not None:
        mk = masks.view(torch.int32) if masks.dtype == torch.uint32 else masks
        if mk.dtype != torch.int32 or mk.shape[0] != M or not mk.is_contiguous():
            raise ValueError("masks must be a contiguous [M, ceil(V/32)] 32-bit tensor")
    od = None
    if order is not None:
        if order.dtype != torch.int32 or order.numel() != M or not order.is_contiguous():
            raise ValueError("order must be a contiguous [M] int32 tensor")
        od = order
    if out is None:
        out = torch.empty((M, Co), dtype=feats.dtype, device=dev)
    if M == 0:
        return out
    before_launch(dev)
    st = status_word(dev)
    if split:
        need = int(lib.spconv_conv_splitk_workspace_bytes(M, Co))
        ws = torch.empty((need,), dtype=torch.uint8, device=dev)
        rc = lib.spconv_submanifold_conv_forward_splitk(
            feats.data_ptr(), DTYPE_CODES[feats.dtype], M, Ci, w.data_ptr(),
            None if b is None else b.data_ptr(), Co, V, nb.data_ptr(),
            None if mk is None else mk.data_ptr(), None if od is None else od.data_ptr(),
            ws.data_ptr(), need, out.data_ptr(), st.word.data_ptr(), _stream_ptr(dev))
        if rc != SPCONV_OK:
            _raise(rc, "spconv_submanifold_conv_forward_splitk")
        return out
    rc = lib.spconv_submanifold_conv_forward_ex(
        feats.data_ptr(), DTYPE_CODES[feats.dtype], M, Ci, w.data_ptr(),
        None if b is None else b.data_ptr(), Co, V, nb.data_ptr(),
        None if mk is None else mk.data_ptr(), None if od is None else od.data_ptr(),
        out.data_ptr(), st.word.data_ptr(), _stream_ptr(dev), int(kernel))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_submanifold_conv_forward")
    return out


def dense_to_sparse(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(indices [M,4] int32 (b,x,y,z), features [M,C]) of the voxels of a channels-last dense
    [B, W, H, D, C] CUDA tensor with any non-zero channel, in (b, x, y, z) order. Reads the
    number of active voxels back to the host (one synchronisation) to size the outputs."""
    lib = load_library()
    dev = _require_cuda(x)
    if x.dtype not in DTYPE_CODES or x.dim() != 5:
        raise ValueError("expected a [B, W, H, D, C] float32/float16/bfloat16 tensor")
    x = x.contiguous()
    B, W, H, D, C = (int(v) for v in x.shape)
    if B * W * H * D == 0 or C == 0:
        return (torch.empty((0, 4), dtype=torch.int32, device=dev),
                torch.empty((0, C), dtype=x.dtype, device=dev))
    need = int(lib.spconv_from_dense_workspace_bytes(B, W, H, D))
    if need <= 0:
        raise ValueError("dense tensor too large")
    ws = torch.empty((need,), dtype=torch.uint8, device=dev)
    count = torch.zeros((1,), dtype=torch.int64, device=dev)
    stream = _stream_ptr(dev)
    rc = lib.spconv_from_dense(x.data_ptr(), DTYPE_CODES[x.dtype], B, W, H, D, C, ws.data_ptr(), need,
                               count.data_ptr(), None, None, 0, 0, stream)
    if rc != SPCONV_OK:
        _raise(rc, "spconv_from_dense")
    M = int(count.item())
    indices = torch.empty((M, 4), dtype=torch.int32, device=dev)
    feats = torch.empty((M, C), dtype=x.dtype, device=dev)
    rc = lib.spconv_from_dense(x.data_ptr(), DTYPE_CODES[x.dtype], B, W, H, D, C, ws.data_ptr(), need,
                               count.data_ptr(), indices.data_ptr(), feats.data_ptr(), M, 1, stream)
    if rc != SPCONV_OK:
        _raise(rc, "spconv_from_dense")
    return indices, feats


def sparse_to_dense(feats: torch.Tensor, indices: torch.Tensor, batch: int, spatial: Sequence[int],
                    channels_first: bool = True) -> torch.Tensor:
    """Zero dense tensor [B, C, W, H, D] (or [B, W, H, D, C]) with the rows of ``feats`` at
    ``indices`` ([M,4] int32 (b,x,y,z))."""
    lib = load_library()
    dev = _require_cuda(feats, indices)
    if feats.dtype not in DTYPE_CODES:
        raise TypeError(f"unsupported feature dtype {feats.dtype}")
    feats = feats.contiguous()
    idx = indices.to(torch.int32).contiguous()
    M, C = int(feats.shape[0]), int(feats.shape[1])
    W, H, D = (int(v) for v in spatial)
    shape = (batch, C, W, H, D) if channels_first else (batch, W, H, D, C)
    out = torch.empty(shape, dtype=feats.dtype, device=dev)
    before_launch(dev)
    st = status_word(dev)
    rc = lib.spconv_to_dense(feats.data_ptr(), DTYPE_CODES[feats.dtype], idx.data_ptr(), M, C, int(batch), W, H, D,
                             1 if channels_first else 0, out.data_ptr(), st.word.data_ptr(), _stream_ptr(dev))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_to_dense")
    return out


_BITS = {torch.uint32: 32, torch.int32: 32, torch.uint64: 64, torch.int64: 64}


def _table_args(table_keys: torch.Tensor, table_values: torch.Tensor, keys: torch.Tensor):
    if table_keys.dtype not in _BITS or table_values.dtype not in _BITS:
        raise TypeError("table keys / values must be 32- or 64-bit integer tensors")
    if keys.dtype != table_keys.dtype:
        raise TypeError(f"keys dtype {keys.dtype} differs from the table's {table_keys.dtype}")
    if not (table_keys.is_contiguous() and table_values.is_contiguous()):
        raise ValueError("table tensors must be contiguous")
    if table_keys.numel() != table_values.numel() or table_keys.numel() == 0:
        raise ValueError("table keys and values must have the same, non-zero length")
    return int(table_keys.numel()), _BITS[table_keys.dtype], _BITS[table_values.dtype]


def hashmap_insert(table_keys: torch.Tensor, table_values: torch.Tensor, keys: torch.Tensor,
                   values: torch.Tensor) -> None:
    """hashmap_insert_cuda (hash.cu:8-71): insert keys -> values into the caller's table."""
    lib = load_library()
    dev = _require_cuda(table_keys, table_values, keys, values)
    cap, kb, vb = _table_args(table_keys, table_values, keys)
    if values.dtype != table_values.dtype or values.numel() != keys.numel():
        raise ValueError("values must match the table's value dtype and the number of keys")
    k, v = keys.contiguous(), values.contiguous()
    before_launch(dev)
    st = status_word(dev)
    rc = lib.spconv_hashmap_insert(table_keys.data_ptr(), table_values.data_ptr(), cap, kb, vb, k.data_ptr(),
                                   v.data_ptr(), int(k.numel()), st.word.data_ptr(), _stream_ptr(dev))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_hashmap_insert")
    after_launch(dev)


def hashmap_lookup(table_keys: torch.Tensor, table_values: torch.Tensor, keys: torch.Tensor) -> torch.Tensor:
    """hashmap_lookup_cuda (hash.cu:73-146): values of keys (all ones if absent)."""
    lib = load_library()
    dev = _require_cuda(table_keys, table_values, keys)
    cap, kb, vb = _table_args(table_keys, table_values, keys)
    k = keys.contiguous()
    out = torch.empty((k.numel(),), dtype=table_values.dtype, device=dev)
    rc = lib.spconv_hashmap_lookup(table_keys.data_ptr(), table_values.data_ptr(), cap, kb, vb, k.data_ptr(),
                                   out.data_ptr(), int(k.numel()), _stream_ptr(dev))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_hashmap_lookup")
    return out


def conv_backward_input(grad_out: torch.Tensor, weight: torch.Tensor, nbr: torch.Tensor,
                        masks: Optional[torch.Tensor], order: Optional[torch.Tensor],
                        nbr_t: Optional[torch.Tensor] = None, masks_t: Optional[torch.Tensor] = None
                        ) -> torch.Tensor:
    """grad_in[j] = sum over (i, v) with nbr[i, v] = j of grad_out[i] @ weight[:, v, :], for
    weight [Co, V, Ci] (or [Co, Kw, Kh, Kd, Ci]). Odd V reads ``nbr`` with the offsets reversed;
    even V needs ``nbr_t`` / ``masks_t`` from ``transpose_neighbor_map``."""
    lib = load_library()
    dev = _require_cuda(grad_out, weight, nbr, masks, order, nbr_t, masks_t)
    if grad_out.dtype not in DTYPE_CODES:
        raise TypeError(f"unsupported dtype {grad_out.dtype}")
    g = grad_out.contiguous()
    M, Co = int(g.shape[0]), int(g.shape[1])
    nb = nbr.view(torch.int32) if nbr.dtype == torch.uint32 else nbr
    V = int(nb.shape[1])
    Ci = int(weight.shape[-1])
    if int(weight.shape[0]) != Co:
        raise ValueError(f"weight has {weight.shape[0]} output channels, grad_out {Co}")
    if V % 2 == 0 and nbr_t is None:
        raise ValueError("an even kernel volume needs the transposed map (transpose_neighbor_map)")
    w_t = weight.reshape(Co, V, Ci).permute(2, 1, 0).to(g.dtype).contiguous()      # [Ci, V, Co]

    def i32(t):
        return None if t is None else (t.view(torch.int32) if t.dtype == torch.uint32 else t)

    def ptr(t):
        return None if t is None else t.data_ptr()
    out = torch.empty((M, Ci), dtype=g.dtype, device=dev)
    if M == 0:
        return out
    before_launch(dev)
    st = status_word(dev)
    rc = lib.spconv_submanifold_conv_backward_input(
        g.data_ptr(), DTYPE_CODES[g.dtype], M, Co, w_t.data_ptr(), Ci, V, nb.data_ptr(), ptr(i32(masks)),
        ptr(order), ptr(i32(nbr_t)), ptr(i32(masks_t)), out.data_ptr(), st.word.data_ptr(), _stream_ptr(dev))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_submanifold_conv_backward_input")
    return out


def transpose_neighbor_map(nbr: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(nbr_t, masks_t): nbr_t[j, v] = i where nbr[i, v] = j (-1 if none), and its offset masks."""
    lib = load_library()
    dev = _require_cuda(nbr)
    nb = nbr.view(torch.int32) if nbr.dtype == torch.uint32 else nbr
    if nb.dtype != torch.int32 or nb.dim() != 2 or not nb.is_contiguous():
        raise ValueError("neighbor map must be a contiguous [M, V] int32/uint32 tensor")
    M, V = int(nb.shape[0]), int(nb.shape[1])
    nbr_t = torch.empty((M, V), dtype=torch.int32, device=dev)
    masks_t = torch.empty((M, mask_words(V)), dtype=torch.int32, device=dev)
    if M == 0:
        return nbr_t, masks_t
    before_launch(dev)
    st = status_word(dev)
    rc = lib.spconv_transpose_neighbor_map(nb.data_ptr(), M, V, nbr_t.data_ptr(), masks_t.data_ptr(),
                                           st.word.data_ptr(), _stream_ptr(dev))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_transpose_neighbor_map")
    return nbr_t, masks_t


def conv_weight_grad(feats: torch.Tensor, grad_out: torch.Tensor, nbr: torch.Tensor,
                     order: Optional[torch.Tensor], with_bias: bool = True,
                     masks: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(grad_weight [Co, V, Ci] fp32, grad_bias [Co] fp32 or None) of the submanifold conv:
    grad_weight[co, v, ci] = sum_i grad_out[i, co] * feats[nbr[i, v], ci]."""
    lib = load_library()
    dev = _require_cuda(feats, grad_out, nbr, order, masks)
    if feats.dtype not in DTYPE_CODES:
        raise TypeError(f"unsupported feature dtype {feats.dtype}")
    if grad_out.dtype != feats.dtype:
        raise TypeError(f"grad_out dtype {grad_out.dtype} differs from feats dtype {feats.dtype}")
    if not (feats.is_contiguous() and grad_out.is_contiguous()):
        raise ValueError("feats and grad_out must be contiguous")
    nb = nbr.view(torch.int32) if nbr.dtype == torch.uint32 else nbr
    if nb.dtype != torch.int32 or nb.dim() != 2 or not nb.is_contiguous():
        raise ValueError("neighbor map must be a contiguous [M, V] int32/uint32 tensor")
    M, Ci = int(feats.shape[0]), int(feats.shape[1])
    Co, V = int(grad_out.shape[1]), int(nb.shape[1])
    if grad_out.shape[0] != M or nb.shape[0] != M:
        raise ValueError("feats, grad_out and neighbor map must have the same number of rows")
    if order is not None and (order.dtype != torch.int32 or order.numel() != M or not order.is_contiguous()):
        raise ValueError("order must be a contiguous [M] int32 tensor")
    mk = None
    if masks is not None:
        mk = masks.view(torch.int32) if masks.dtype == torch.uint32 else masks
        if mk.dtype != torch.int32 or mk.shape[0] != M or not mk.is_contiguous():
            raise ValueError("masks must be a contiguous [M, ceil(V/32)] 32-bit tensor")
    gw = torch.empty((Co, V, Ci), dtype=torch.float32, device=dev)
    gb = torch.empty((Co,), dtype=torch.float32, device=dev) if with_bias else None
    ws_bytes = int(lib.spconv_weight_grad_workspace_bytes(M, V))
    ws = torch.empty((max(ws_bytes, 16) + 15) // 16 * 16, dtype=torch.uint8, device=dev)
    before_launch(dev)
    st = status_word(dev)
    rc = lib.spconv_submanifold_conv_weight_grad(
        feats.data_ptr(), grad_out.data_ptr(), DTYPE_CODES[feats.dtype], M, Ci, Co, V, nb.data_ptr(),
        None if mk is None else mk.data_ptr(), None if order is None else order.data_ptr(), gw.data_ptr(),
        None if gb is None else gb.data_ptr(), ws.data_ptr(), ws.numel(), st.word.data_ptr(), _stream_ptr(dev))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_submanifold_conv_weight_grad")
    return gw, gb


def _on_device(fn):
    """Runs a call with the device of its tensors current (launches go to that device's stream)."""
    @functools.wraps(fn)
    def call(first, *args, **kwargs):
        t = first if isinstance(first, torch.Tensor) else first[0]
        index = t.get_device()
        if index < 0 or index == torch._C._cuda_getDevice():
            return fn(first, *args, **kwargs)
        with torch.cuda.device(index):
            return fn(first, *args, **kwargs)
    return call


def _raw_stream(index: int) -> int:
    """The device's current stream, without building a torch.cuda.Stream."""
    return torch._C._cuda_getCurrentRawStream(index)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _matrix(t: torch.Tensor, shape: Tuple[int, ...], dtype: torch.dtype, what: str) -> None:
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{what} dtype {t.dtype} differs from the features' {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


@_on_device
def linear_forward(feats: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                   residual: Optional[torch.Tensor], activation: str, keep_preact: bool = False,
                   kernel: int = KERNEL_AUTO) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(residual + act(feats @ weight.T + bias), act's argument if ``keep_preact``); the bias in fp32 or
    the features' dtype."""
    dev = _require_cuda(feats, weight, bias, residual)
    dtype = feats.dtype
    if dtype not in DTYPE_CODES:
        raise TypeError(f"unsupported feature dtype {dtype}")
    if feats.dim() != 2 or weight.dim() != 2:
        raise ValueError("feats must be [M, Ci] and weight [Co, Ci]")
    if not feats.is_contiguous():
        raise ValueError("feats must be contiguous")
    if activation not in ACTIVATIONS:
        raise ValueError(f"Unsupported activation {activation}.")
    M, Ci = feats.shape
    Co = weight.shape[0]
    if weight.shape[1] != Ci:
        raise ValueError(f"weight has {weight.shape[1]} input channels, feats {Ci}")
    weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
        _matrix(bias, (Co,), torch.float32 if bias.dtype == torch.float32 else dtype, "bias")
    if residual is not None:
        _matrix(residual, (M, Co), dtype, "residual")
    out = torch.empty((M, Co), dtype=dtype, device=dev)
    preact = torch.empty_like(out) if keep_preact else None
    if M == 0:
        return out, preact
    index = dev.index
    lib = _lib or load_library()
    ws, need = None, 0
    if Ci % 8 or Co % 8:
        need = lib.spconv_linear_forward_workspace_bytes(DTYPE_CODES[dtype], M, Ci, Co, residual is not None, keep_preact)
        ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need > 0 else None
    rc = lib.spconv_linear_forward_ex(
        feats.data_ptr(), DTYPE_CODES[dtype], M, Ci, weight.data_ptr(), _ptr(bias),
        0 if bias is None else DTYPE_CODES[bias.dtype], _ptr(residual), Co,
        ACTIVATIONS[activation], out.data_ptr(), _ptr(preact), _ptr(ws), need, kernel, mapped_status(index),
        _raw_stream(index))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_linear_forward_ex")
    after_mapped_launch(index)
    return out, preact


@_on_device
def linear_backward(grad_out: torch.Tensor, preact: Optional[torch.Tensor], feats: torch.Tensor, weight: torch.Tensor,
                    activation: str, weight_dtype: torch.dtype, bias_dtype: Optional[torch.dtype],
                    needs: Sequence[bool], kernel: int = KERNEL_AUTO) -> tuple:
    """Gradients of feats, weight (in ``weight_dtype``) and bias (in ``bias_dtype``), None where
    ``needs`` says so; the arguments are linear_forward's, with its kept product."""
    _require_cuda(grad_out, preact, feats, weight)
    _matrix(grad_out, (feats.shape[0], weight.shape[0]), feats.dtype, "grad_out")
    return linear_backward_of(grad_out, preact, feats, weight.contiguous(), ACTIVATIONS[activation], weight_dtype,
                              bias_dtype, needs, kernel)


def linear_backward_of(grad_out, preact, feats, weight, activation: int, weight_dtype, bias_dtype, needs,
                       kernel: int = KERNEL_AUTO) -> tuple:
    """linear_backward of tensors that a forward has checked (autograd's), contiguous; a network's
    backward calls it once a layer, so it does no more than it must."""
    lib = _lib or load_library()
    M, Ci = feats.shape
    Co = weight.shape[0]
    dtype, dev, index = feats.dtype, feats.device, feats.get_device()
    code = DTYPE_CODES[dtype]
    gx = gw = gb = None
    gx_ptr = gw_ptr = gb_ptr = None
    gw_code = gb_code = 0
    if needs[0]:
        gx = torch.empty_like(feats)
        gx_ptr = gx.data_ptr()
    if needs[1]:                             # in the wanted dtype where the kernels write it
        gw = torch.empty((Co, Ci), dtype=dtype if weight_dtype == dtype else torch.float32, device=dev)
        gw_ptr, gw_code = gw.data_ptr(), code if weight_dtype == dtype else 0
    if needs[2]:
        gb = torch.empty((Co,), dtype=dtype if bias_dtype == dtype else torch.float32, device=dev)
        gb_ptr, gb_code = gb.data_ptr(), code if bias_dtype == dtype else 0
    need = lib.spconv_linear_backward_workspace_bytes(code, M, Ci, Co, activation)
    ws = torch.empty((need if need > 0 else 256,), dtype=torch.uint8, device=dev)
    rc = lib.spconv_linear_backward(
        grad_out.data_ptr(), None if preact is None else preact.data_ptr(), feats.data_ptr(), weight.data_ptr(), code,
        M, Ci, Co, activation, gx_ptr, gw_ptr, gw_code, gb_ptr, gb_code, ws.data_ptr(), need, kernel,
        mapped_status(index), _raw_stream(index))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_linear_backward")
    after_mapped_launch(index)
    if gw is not None and gw.dtype != weight_dtype:
        gw = gw.to(weight_dtype)
    if gb is not None and gb.dtype != bias_dtype:
        gb = gb.to(bias_dtype)
    return gx, gw, gb


def _norm_args(feats: torch.Tensor, residual, params, offsets, residual_scale: float, norm: str,
               next_norm: str, eps: float) -> ResidualNormArgs:
    """Checked arguments shared by the forward and the backward; ``params`` are the gate, weight,
    bias, next_weight and next_bias (each None, [C] or [samples, C])."""
    dev = _require_cuda(feats, residual, *params, offsets)
    if feats.dtype not in DTYPE_CODES:
        raise TypeError(f"unsupported feature dtype {feats.dtype}")
    if feats.dim() != 2 or feats.shape[1] < 1:
        raise ValueError(f"feats must be an [M, C] tensor, got shape {list(feats.shape)}")
    if not feats.is_contiguous():
        raise ValueError("feats must be contiguous")
    if norm not in NORMS or next_norm not in NORMS:
        raise ValueError(f"unsupported norm {norm if norm not in NORMS else next_norm}")
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    M, C = feats.shape
    a = ResidualNormArgs(dtype=DTYPE_CODES[feats.dtype], channels=C, num_rows=M, feats=feats.data_ptr(),
                         num_samples=1, norm=NORMS[norm], next_norm=NORMS[next_norm],
                         residual_scale=residual_scale, eps=eps)
    if residual is not None:
        _matrix(residual, feats.shape, feats.dtype, "residual")
        a.residual = residual.data_ptr()
    per_sample = False
    for name, p in zip(("gate", "weight", "bias", "next_weight", "next_bias"), params):
        if p is None:
            continue
        if (name in ("weight", "bias") and norm == "none") or (name[:5] == "next_" and next_norm == "none"):
            raise ValueError(f"{name} given without its norm")
        if p.dtype != torch.float32 and p.dtype != feats.dtype:
            raise TypeError(f"{name} must be float32 or {feats.dtype}, got {p.dtype}")
        if not p.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if p.dim() == 2:
            if offsets is None:
                raise ValueError(f"{name} has a row per sample: batch_offsets is needed")
            if tuple(p.shape) != (offsets.numel() - 1, C):
                raise ValueError(f"{name} must have shape {[offsets.numel() - 1, C]}, got {list(p.shape)}")
            per_sample = True
        elif p.dim() != 1 or p.shape[0] != C:
            raise ValueError(f"{name} must have shape [{C}] or [samples, {C}], got {list(p.shape)}")
        q = getattr(a, name)
        q.data, q.dtype, q.per_sample = p.data_ptr(), DTYPE_CODES[p.dtype], p.dim() == 2
    if offsets is not None:
        if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() < 2 or not offsets.is_contiguous():
            raise ValueError("batch_offsets must be a contiguous [samples + 1] int32 tensor")
        if per_sample:
            a.offsets, a.num_samples = offsets.data_ptr(), offsets.numel() - 1
    a.status = mapped_status(dev.index)
    return a


@_on_device
def residual_norm_forward(feats: torch.Tensor, residual: Optional[torch.Tensor], params: Sequence[Optional[torch.Tensor]],
                          offsets: Optional[torch.Tensor], residual_scale: float, norm: str, next_norm: str,
                          eps: float, keep_stats: bool = False) -> tuple:
    """(hidden, normed) of the gated residual step (normed None without ``next_norm``); with
    ``keep_stats`` also the row statistics and the call's arguments, for residual_norm_backward_of."""
    a = _norm_args(feats, residual, params, offsets, residual_scale, norm, next_norm, eps)
    hidden = torch.empty_like(feats)
    a.hidden = hidden.data_ptr()
    normed = stats = None
    if next_norm != "none":
        normed = torch.empty_like(feats)
        a.normed = normed.data_ptr()
    if keep_stats:
        stats = torch.empty((a.num_rows, 4), dtype=torch.float32, device=feats.device)
        a.row_stats = stats.data_ptr()
    index = feats.get_device()
    rc = (_lib or load_library()).spconv_residual_norm_forward(a, _raw_stream(index))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_residual_norm_forward")
    after_mapped_launch(index)
    return (hidden, normed, stats, a) if keep_stats else (hidden, normed)


@_on_device
def residual_norm_backward(feats: torch.Tensor, residual: Optional[torch.Tensor], params: Sequence[Optional[torch.Tensor]],
                           offsets: Optional[torch.Tensor], residual_scale: float, norm: str, next_norm: str,
                           eps: float, stats: torch.Tensor, grad_hidden: Optional[torch.Tensor],
                           grad_normed: Optional[torch.Tensor], needs: Sequence[bool]) -> list:
    """Gradients of feats, residual, gate, weight, bias, next_weight and next_bias (None where
    ``needs`` says so), each in its tensor's shape and dtype."""
    a = _norm_args(feats, residual, params, offsets, residual_scale, norm, next_norm, eps)
    for g, what in ((grad_hidden, "grad_hidden"), (grad_normed, "grad_normed")):
        if g is not None:
            _require_cuda(feats, g)
            _matrix(g, feats.shape, feats.dtype, what)
    return residual_norm_backward_of(a, feats, residual, params, offsets, stats, grad_hidden, grad_normed, needs)


def residual_norm_backward_of(args: ResidualNormArgs, feats, residual, params, offsets, stats, grad_hidden, grad_normed,
                              needs) -> list:
    """residual_norm_backward with the arguments that a forward of the same tensors has checked: only
    the addresses are taken anew (saved tensors may have been moved)."""
    lib, index = _lib or load_library(), feats.get_device()
    a = ResidualNormArgs.from_buffer_copy(args)
    a.hidden = a.normed = None
    a.feats, a.row_stats = feats.data_ptr(), stats.data_ptr()
    a.grad_hidden = None if grad_hidden is None else grad_hidden.data_ptr()
    a.grad_normed = None if grad_normed is None else grad_normed.data_ptr()
    grads = [None] * 7
    if needs[0]:
        grads[0] = g = torch.empty_like(feats)
        a.grad_feats = g.data_ptr()
    if residual is not None:
        a.residual = residual.data_ptr()
        if needs[1]:
            grads[1] = g = torch.empty_like(residual)
            a.grad_residual = g.data_ptr()
    sums = False
    for i, (q, p) in enumerate(zip((a.gate, a.weight, a.bias, a.next_weight, a.next_bias), params), 2):
        if p is not None:
            q.data = p.data_ptr()
            if needs[i]:
                grads[i] = g = torch.empty_like(p)
                q.grad = g.data_ptr()
                sums = True
    if a.offsets:
        a.offsets = offsets.data_ptr()
    if sums:
        a.workspace_bytes = need = lib.spconv_residual_norm_workspace_bytes(a.num_rows, a.channels, a.num_samples)
        ws = torch.empty((need,), dtype=torch.uint8, device=feats.device)
        a.workspace = ws.data_ptr()
    a.status = mapped_status(index)
    rc = lib.spconv_residual_norm_backward(a, _raw_stream(index))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_residual_norm_backward")
    after_mapped_launch(index)
    return grads


_data_ptr, _numel, _get_device, _is_contiguous = (
    getattr(torch.Tensor, name) for name in ("data_ptr", "numel", "get_device", "is_contiguous"))
_dtype = operator.attrgetter("dtype")


def _is_dense(t: torch.Tensor) -> bool:
    """Whether the elements fill their memory without gaps or overlap, in any order of dimensions."""
    if t.is_contiguous():
        return True
    order = sorted(range(t.dim()), key=lambda d: (t.stride(d), t.size(d)), reverse=True)
    return t.permute(order).is_contiguous()


@_on_device
def clip_gradients(grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor], max_norm: float,
                   norm_kind: int) -> torch.Tensor:
    """outs[k] = grads[k] * min(1, max_norm / (norm + 1e-6)); returns the norm (0-dim float32)."""
    lib = load_library()
    dev, index = grads[0].device, grads[0].get_device()
    n = len(grads)
    # whole lists at a time: a network has hundreds of gradients
    ptrs, sizes, dtypes = (list(map(f, grads)) for f in (_data_ptr, _numel, _dtype))
    where = set(map(_get_device, grads))
    optrs = ptrs
    if outs is not grads:
        optrs = list(map(_data_ptr, outs))
        where.update(map(_get_device, outs))
        if list(map(_numel, outs)) != sizes or list(map(_dtype, outs)) != dtypes:
            raise ValueError("each output must have its gradient's size and dtype")
    if where != {index} or index < 0:
        _require_cuda(*grads, *outs)
    if not (all(map(_is_contiguous, grads)) and (outs is grads or all(map(_is_contiguous, outs)))):
        for g, o in zip(grads, outs):
            if not _is_dense(g):
                raise ValueError("gradients must be dense in memory")
            if o.stride() != g.stride() and not (g.is_contiguous() and o.is_contiguous()):
                raise ValueError("each output must have its gradient's strides")
    try:
        codes = [DTYPE_CODES[d] for d in dtypes]
    except KeyError as e:
        raise TypeError(f"unsupported gradient dtype {e.args[0]}") from None
    ptrs, optrs, sizes, codes = (array.array(t, v) for t, v in (("Q", ptrs), ("Q", optrs), ("q", sizes), ("i", codes)))
    mapped_status(index)                     # a step's gradients end here: what went wrong on the way is raised
    total = torch.empty((), dtype=torch.float32, device=dev)
    need = lib.spconv_clip_gradients_workspace_bytes(n)
    ws = torch.empty((need,), dtype=torch.uint8, device=dev)
    rc = lib.spconv_clip_gradients(ptrs.buffer_info()[0], optrs.buffer_info()[0], sizes.buffer_info()[0],
                                   codes.buffer_info()[0], n, norm_kind, max_norm, total.data_ptr(),
                                   ws.data_ptr(), need, _raw_stream(index))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_clip_gradients")
    # written through their addresses: a backward that saved them has to notice
    torch.autograd.graph.increment_version(outs)
    after_mapped_launch(index)
    return total


def set_wait_limit_ns(limit_ns: int) -> int:
    """Time limit of the pipeline waits inside the tensor-core conv kernels launched from now
    on (process-wide; 0 restores the 2 s default). Returns the previous limit. A kernel whose
    wait reaches it abandons its work and reports SPCONV_STATUS_WAIT_TIMEOUT."""
    return int(load_library().spconv_set_wait_limit_ns(int(limit_ns)))


def stage_timing(max_calls: int) -> None:
    """Start (max_calls > 0) or stop (0) per-stage device timing inside the library."""
    rc = load_library().spconv_stage_timing(int(max_calls))
    if rc != SPCONV_OK:
        _raise(rc, "spconv_stage_timing")


def stage_times_ms() -> dict:
    """{stage: (summed ms, launches)} for the calls recorded since stage_timing(n)."""
    import numpy as np
    ms = np.zeros(len(STAGES), dtype=np.float64)
    cnt = np.zeros(len(STAGES), dtype=np.int64)
    n = load_library().spconv_stage_times_ms(ms.ctypes.data, cnt.ctypes.data, len(STAGES))
    if n < 0:
        _raise(SPCONV_ERR_CUDA, "spconv_stage_times_ms")
    return {STAGES[i]: (float(ms[i]), int(cnt[i])) for i in range(n)}
