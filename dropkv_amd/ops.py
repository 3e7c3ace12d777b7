"""Torch-tensor wrappers around the C ABI of libdropkv_amd.so.

PyTorch provides device memory (its caching allocator, also for the
workspaces) and the current HIP stream; all arithmetic runs in the HIP
kernels.  The wrappers check what the kernels assume (device, dtype, layout,
alignment) and raise ``RuntimeError`` otherwise; the reference-compatible
``AssertionError`` guards live in :mod:`dropkv_amd.dropkv_triton`.
"""

from __future__ import annotations

import functools
import threading
from typing import NamedTuple, Optional

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib

_DTYPE_CODE = {torch.bfloat16: _lib.DROPKV_BF16, torch.float16: _lib.DROPKV_FP16, torch.float32: _lib.DROPKV_FP32}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev: torch.device) -> int:
    """The current stream of ``dev`` as a raw handle (the raw getter takes
    ~0.1 us where building a torch Stream object takes ~2 us per call)."""
    if _raw_stream is not None and dev.index is not None:
        return _raw_stream(dev.index)
    return torch.cuda.current_stream(dev).cuda_stream


def _workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=dev)


def _evict_workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    """A new ``dropkv_scores`` / ``dropkv_evict`` workspace: its leading
    counters (_lib.SYNC_BYTES) start at zero, and every call leaves them zero."""
    ws = _workspace(nbytes, dev)
    ws[: _lib.SYNC_BYTES].zero_()
    return ws


# One workspace per (device, stream, thread), grown on demand and reused by every
# call of that thread on that stream that brings none: the kernels of one
# thread's calls run in order, so they never use it at the same time.  (Two
# threads' calls on one stream may put their kernels between one another's.)  A
# thread's go back to the allocator when it ends.
_shared_ws: dict = {}
_shared_ws_lock = threading.RLock()  # (an ended thread's mark may go in a collection under the lock)


class _ThreadMark:
    """Lives as long as its thread, whose workspaces go with it."""

    def __init__(self):
        self.ident = threading.get_ident()

    def __del__(self):
        if _shared_ws_lock is None:  # (the interpreter is ending)
            return
        with _shared_ws_lock:
            for key in list(_shared_ws or ()):
                if key[-1] == self.ident:
                    _shared_ws.pop(key, None)


_thread_local = threading.local()


def _stream_workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    nbytes = max(int(nbytes), 1)
    if torch.cuda.is_current_stream_capturing():
        return _evict_workspace(nbytes, dev)  # a graph keeps its own (private-pool) workspace
    key = (dev.index, _stream(dev), threading.get_ident())
    with _shared_ws_lock:
        ws = _shared_ws.get(key)
        if ws is None or ws.numel() < nbytes:
            if not hasattr(_thread_local, "mark"):
                _thread_local.mark = _ThreadMark()
            ws = _evict_workspace(nbytes, dev)
            _shared_ws[key] = ws
    return ws


def release_workspaces() -> None:
    """Drop the per-(device, stream, thread) workspaces kept for calls that bring
    none (they only grow, to the largest call seen there, and are otherwise
    held for the life of their thread).  Each goes back to
    PyTorch's caching allocator, which orders its reuse after the work
    already enqueued on its stream (``torch.cuda.empty_cache()`` can then
    return it to the device); the next call allocates a fresh workspace."""
    with _shared_ws_lock:
        _shared_ws.clear()


def _aligned(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0


def _kv_operand(t: torch.Tensor) -> torch.Tensor:
    """K/V must be contiguous and 16-byte aligned for the vector loads."""
    if not t.is_contiguous() or not _aligned(t):
        t = t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def _evict_kv(t: torch.Tensor):
    """``t`` (K or V, [B, H, L, D]) as the layer-call reads it, and its
    (batch, head, row) element strides: in place where its rows are whole
    16-byte units apart and do not overlap (a decoder layer's [B, L, H, D]
    projection seen as [B, H, L, D], say), else a dense copy.  The rule is
    that of ``dropkv_evict_strided``."""
    B, H, L, D = t.shape
    dense = (H * L * D, L * D, D)
    if t.is_contiguous():
        return (t if _aligned(t) else t.clone()), dense
    sb, sh, sl, sd = t.stride()
    es = t.element_size()
    if (sd == 1 and sl >= D and ((sb | sh | sl | D) * es) % 16 == 0 and _aligned(t)
            and sl <= (1 << 31) // es // (L + 1024)):
        return t, (sb, sh, sl)
    return t.contiguous(), dense


def _check_device(*ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    if dev.type != "cuda":
        raise RuntimeError("DropKV HIP ops need tensors on a ROCm (cuda) device")
    for t in ts[1:]:
        if t.device != dev:
            raise RuntimeError("all tensors must be on the same device")
    return dev


def scores(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, eps: float = 1e-6,
           p_round: bool = True, y_round: bool = False, splits: int = 0,
           return_workspace: bool = False):
    """Per-key DropKV scores [B, Hkv, Lk] fp32 (see ``dropkv_scores`` in the C ABI)."""
    dev = _check_device(Q, K, V)
    if Q.dtype not in _DTYPE_CODE or K.dtype != Q.dtype or V.dtype != Q.dtype:
        raise RuntimeError(f"unsupported dtype combination {Q.dtype}/{K.dtype}/{V.dtype}")
    B, Hq, Lq, D = Q.shape
    Hkv, Lk = K.shape[1], K.shape[2]
    K = _kv_operand(K)
    V = _kv_operand(V)
    lib = _lib.load()
    ws_bytes = lib.dropkv_scores_workspace_bytes(B, Hq, Hkv, Lk, D, window, splits)
    ws = _evict_workspace(ws_bytes, dev) if return_workspace else _stream_workspace(ws_bytes, dev)
    out = torch.empty(B, Hkv, Lk, dtype=torch.float32, device=dev)
    rc = lib.dropkv_scores(Q.data_ptr(), *Q.stride(), K.data_ptr(), V.data_ptr(), _DTYPE_CODE[Q.dtype],
                           B, Hq, Hkv, Lq, Lk, D, window, float(eps), int(bool(p_round)), int(bool(y_round)),
                           int(splits), out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(dev))
    _lib.check(rc, "dropkv_scores")
    if return_workspace:
        return out, ws
    return out


def scores_debug_state(ws: torch.Tensor, B: int, Hq: int, Hkv: int, Lk: int, D: int, window: int,
                       splits: int = 0):
    """(lse [B,Hkv,M] natural log, y [B,Hkv,M,D] fp32) left in a scoring workspace."""
    dev = ws.device
    M = (Hq // Hkv) * window
    lse = torch.empty(B, Hkv, M, dtype=torch.float32, device=dev)
    y = torch.empty(B, Hkv, M, D, dtype=torch.float32, device=dev)
    rc = _lib.load().dropkv_scores_debug_state(ws.data_ptr(), B, Hq, Hkv, Lk, D, window, splits,
                                               lse.data_ptr(), y.data_ptr(), _stream(dev))
    _lib.check(rc, "dropkv_scores_debug_state")
    return lse, y


def select(scores_t: torch.Tensor, kernel_size: int, window: int, keep: int, return_pooled: bool = False):
    """Pool, protect, top-k and sort: int64 indices [..., keep], ascending."""
    dev = _check_device(scores_t)
    if scores_t.dtype != torch.float32:
        raise RuntimeError("select expects fp32 scores")
    s = scores_t.contiguous()
    Lk = s.shape[-1]
    rows = s.numel() // Lk
    lib = _lib.load()
    ws = _workspace(lib.dropkv_select_workspace_bytes(rows, Lk), dev)
    idx = torch.empty(*s.shape[:-1], keep, dtype=torch.int64, device=dev)
    pooled = torch.empty_like(s) if return_pooled else None
    rc = lib.dropkv_select(s.data_ptr(), rows, Lk, kernel_size, window, keep, idx.data_ptr(),
                           pooled.data_ptr() if pooled is not None else None, ws.data_ptr(), ws.numel(),
                           _stream(dev))
    _lib.check(rc, "dropkv_select")
    if return_pooled:
        return idx, pooled
    return idx


def _seg_strides(t: torch.Tensor):
    if t.stride(3) != 1:
        raise RuntimeError("the head-dim axis of K/V must be contiguous")
    return t.stride(0), t.stride(1), t.stride(2)


def compact(K: torch.Tensor, V: torch.Tensor, idx: torch.Tensor):
    """Bit-exact gather of rows ``idx`` [B,H,keep] from K/V [B,H,L,D]."""
    dev = _check_device(K, V, idx)
    if K.shape != V.shape or K.stride() != V.stride() or K.dtype != V.dtype:
        raise RuntimeError("K and V must have the same shape, strides and dtype")
    if K.stride(3) != 1:
        K, V = K.contiguous(), V.contiguous()
    idx = idx.to(torch.int64).contiguous()
    B, H, L, D = K.shape
    keep = idx.shape[-1]
    ko = torch.empty(B, H, keep, D, dtype=K.dtype, device=dev)
    vo = torch.empty_like(ko)
    rc = _lib.load().dropkv_compact(K.data_ptr(), V.data_ptr(), *_seg_strides(K), K.element_size(), B, H, L, D,
                                    idx.data_ptr(), keep, ko.data_ptr(), vo.data_ptr(), _stream(dev))
    _lib.check(rc, "dropkv_compact")
    return ko, vo


def compact2(K0: torch.Tensor, V0: torch.Tensor, K1: torch.Tensor, V1: torch.Tensor, idx: torch.Tensor):
    """Gather from the logical concatenation [K0 | K1] along the sequence axis."""
    dev = _check_device(K0, V0, K1, V1, idx)
    if K0.stride(3) != 1 or V0.stride(3) != 1:
        K0, V0 = K0.contiguous(), V0.contiguous()
    if K1.stride(3) != 1 or V1.stride(3) != 1:
        K1, V1 = K1.contiguous(), V1.contiguous()
    if K0.stride() != V0.stride() or K1.stride() != V1.stride():
        K0, V0, K1, V1 = K0.contiguous(), V0.contiguous(), K1.contiguous(), V1.contiguous()
    idx = idx.to(torch.int64).contiguous()
    B, H, L0, D = K0.shape
    L1 = K1.shape[2]
    keep = idx.shape[-1]
    ko = torch.empty(B, H, keep, D, dtype=K0.dtype, device=dev)
    vo = torch.empty_like(ko)
    rc = _lib.load().dropkv_compact2(K0.data_ptr(), V0.data_ptr(), *_seg_strides(K0), L0,
                                     K1.data_ptr(), V1.data_ptr(), *_seg_strides(K1), L1,
                                     K0.element_size(), B, H, D, idx.data_ptr(), keep, ko.data_ptr(),
                                     vo.data_ptr(), _stream(dev))
    _lib.check(rc, "dropkv_compact2")
    return ko, vo


def _check_buffer(buf: torch.Tensor, name: str):
    if buf.dim() != 4 or not buf.is_contiguous() or not _aligned(buf):
        raise RuntimeError(f"{name} must be a contiguous, 16-byte aligned [B, H, capacity, D] buffer")


def append(K: torch.Tensor, V: torch.Tensor, k_buf: torch.Tensor, v_buf: torch.Tensor, row0: int):
    """Copy K/V [B, H, L, D] (any strides, head dim contiguous) bit for bit
    to rows ``row0 .. row0+L-1`` of the [B, H, capacity, D] buffers
    (``dropkv_append``)."""
    dev = _check_device(K, V, k_buf, v_buf)
    _check_buffer(k_buf, "k_buf")
    _check_buffer(v_buf, "v_buf")
    # (Shapes and strides read once: this call runs per layer and chunk, and
    # its host time is of the order of the copy's.)
    shape, bshape, dtype = K.shape, k_buf.shape, K.dtype
    if shape != V.shape or dtype != V.dtype or bshape != v_buf.shape:
        raise RuntimeError("K/V and the buffers must match in shape and dtype")
    B, H, L, D = shape
    bB, bH, C, bD = bshape
    if dtype != k_buf.dtype or B != bB or H != bH or D != bD:
        raise RuntimeError("K/V do not fit the buffers")
    strides = K.stride()
    if strides[3] != 1 or strides != V.stride():
        K, V = K.contiguous(), V.contiguous()
        strides = K.stride()
    rc = _lib.load().dropkv_append(K.data_ptr(), V.data_ptr(), strides[0], strides[1], strides[2], K.element_size(),
                                   B, H, L, D, k_buf.data_ptr(), v_buf.data_ptr(), C, int(row0), _stream(dev))
    _lib.check(rc, "dropkv_append")


def evict_ld(Q: torch.Tensor, k_buf: torch.Tensor, v_buf: torch.Tensor, Lk: int, window: int, kernel_size: int,
             keep: int, k_out: torch.Tensor, v_out: torch.Tensor, protect_window: int | None = None,
             eps: float = 1e-6, p_round: bool = True, y_round: bool = False) -> torch.Tensor:
    """One layer-call (``dropkv_evict_ld``) on K/V held in rows 0 .. Lk-1 of
    [B, Hkv, capacity, D] buffers, writing the compressed rows to rows
    0 .. keep-1 of the ``k_out`` / ``v_out`` buffers.  Returns the kept
    indices [B, Hkv, keep] (ascending)."""
    dev = _check_device(Q, k_buf, v_buf, k_out, v_out)
    for t, n in ((k_buf, "k_buf"), (v_buf, "v_buf"), (k_out, "k_out"), (v_out, "v_out")):
        _check_buffer(t, n)
    if Q.dtype not in _DTYPE_CODE or k_buf.dtype != Q.dtype or v_buf.dtype != Q.dtype or k_out.dtype != Q.dtype:
        raise RuntimeError("Q, the K/V buffers and the outputs must share a bf16/fp16 dtype")
    if k_buf.shape != v_buf.shape or k_out.shape != v_out.shape:
        raise RuntimeError("K and V buffers must have the same shape")
    B, Hq, Lq, D = Q.shape
    Hkv = k_buf.shape[1]
    lib = _lib.load()
    ws = _stream_workspace(lib.dropkv_evict_workspace_bytes(B, Hq, Hkv, Lk, D, window, 0), dev)
    idx = torch.empty(B, Hkv, keep, dtype=torch.int64, device=dev)
    pw = window if protect_window is None else protect_window
    rc = lib.dropkv_evict_ld(Q.data_ptr(), *Q.stride(), k_buf.data_ptr(), v_buf.data_ptr(), k_buf.shape[2],
                             _DTYPE_CODE[Q.dtype], B, Hq, Hkv, Lq, int(Lk), D, int(window), float(eps),
                             int(bool(p_round)), int(bool(y_round)), 0, int(kernel_size), int(pw), int(keep), None,
                             idx.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), k_out.shape[2], ws.data_ptr(),
                             ws.numel(), _stream(dev))
    _lib.check(rc, "dropkv_evict_ld")
    return idx


def evict(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, kernel_size: int, keep: int,
          protect_window: int | None = None, eps: float = 1e-6, p_round: bool = True, y_round: bool = False,
          splits: int = 0):
    """One layer-call (``dropkv_evict``): score, pool, protect, top-k, sort and
    gather in one call.  Returns fresh ``(keep_idx [B,Hkv,keep] int64,
    k_out, v_out [B,Hkv,keep,D])``, like the reference's
    ``_compute_keep_indices`` + ``_gather_compressed``; the workspace is the
    current stream's shared one."""
    dev = _check_device(Q, K, V)
    if Q.dtype not in _DTYPE_CODE or K.dtype != Q.dtype or V.dtype != Q.dtype:
        raise RuntimeError(f"unsupported dtype combination {Q.dtype}/{K.dtype}/{V.dtype}")
    if K.shape != V.shape:
        raise RuntimeError("K and V must have the same shape")
    B, Hq, Lq, D = Q.shape
    Hkv, Lk = K.shape[1], K.shape[2]
    K, k_strides = _evict_kv(K)
    V, v_strides = _evict_kv(V)
    lib = _lib.load()
    ws = _stream_workspace(lib.dropkv_evict_workspace_bytes(B, Hq, Hkv, Lk, D, window, splits), dev)
    idx = torch.empty(B, Hkv, keep, dtype=torch.int64, device=dev)
    ko = torch.empty(B, Hkv, keep, D, dtype=Q.dtype, device=dev)
    vo = torch.empty_like(ko)
    pw = window if protect_window is None else protect_window
    rc = lib.dropkv_evict_strided(Q.data_ptr(), *Q.stride(), K.data_ptr(), *k_strides, V.data_ptr(), *v_strides,
                                  _DTYPE_CODE[Q.dtype], B, Hq, Hkv, Lq, Lk, D, int(window), float(eps),
                                  int(bool(p_round)), int(bool(y_round)), int(splits), int(kernel_size), int(pw),
                                  int(keep), None, idx.data_ptr(), ko.data_ptr(), vo.data_ptr(), int(keep),
                                  ws.data_ptr(), ws.numel(), _stream(dev))
    _lib.check(rc, "dropkv_evict")
    return idx, ko, vo


def set_tail_select(enabled: bool = True, spin_polls: int = -1, spin_polls_b: int = -1) -> None:
    """``dropkv_set_tail_select``: whether layer-calls finish their selection
    (threshold, ordered emit, K/V gather) in the scoring kernel's tail when
    the call allows it (on by default) or always in two further kernels; the
    polls a workgroup waits at the tail's first barrier before it leaves its
    row to the last one to arrive (``spin_polls``), and at the second barrier
    before it finishes the row alone (``spin_polls_b``); < 0 leaves a limit
    unchanged, 0 forces that path.  Same results every way."""
    _lib.check(_lib.load().dropkv_set_tail_select(int(bool(enabled)), int(spin_polls), int(spin_polls_b)),
               "dropkv_set_tail_select")


class EvictPlan:
    """Pre-sized workspace and outputs for repeated layer-calls of one shape
    (``dropkv_evict``); avoids per-call allocation in tight loops."""

    def __init__(self, Q: torch.Tensor, K: torch.Tensor, window: int, kernel_size: int, keep: int,
                 protect_window: int | None = None, eps: float = 1e-6, p_round: bool = True,
                 y_round: bool = False, splits: int = 0, keep_scores: bool = False):
        dev = _check_device(Q, K)
        B, Hq, Lq, D = Q.shape
        Hkv, Lk = K.shape[1], K.shape[2]
        self.shape = (B, Hq, Hkv, Lq, Lk, D)
        self.dtype = Q.dtype
        self.window, self.kernel_size, self.keep = int(window), int(kernel_size), int(keep)
        self.protect_window = int(window if protect_window is None else protect_window)
        self.eps, self.p_round, self.y_round, self.splits = float(eps), int(p_round), int(y_round), int(splits)
        lib = _lib.load()
        self.ws = _evict_workspace(lib.dropkv_evict_workspace_bytes(B, Hq, Hkv, Lk, D, window, splits), dev)
        self.scores = torch.empty(B, Hkv, Lk, dtype=torch.float32, device=dev) if keep_scores else None
        self.keep_idx = torch.empty(B, Hkv, keep, dtype=torch.int64, device=dev)
        self.k_out = torch.empty(B, Hkv, keep, D, dtype=Q.dtype, device=dev)
        self.v_out = torch.empty_like(self.k_out)
        self.dev = dev

    def __call__(self, Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor):
        B, Hq, Hkv, Lq, Lk, D = self.shape
        if tuple(Q.shape) != (B, Hq, Lq, D) or tuple(K.shape) != (B, Hkv, Lk, D) or K.shape != V.shape:
            raise RuntimeError("input shapes differ from the plan")
        if Q.dtype != self.dtype or K.dtype != self.dtype or V.dtype != self.dtype:
            raise RuntimeError("input dtype differs from the plan")
        K, k_strides = _evict_kv(K)
        V, v_strides = _evict_kv(V)
        rc = _lib.load().dropkv_evict_strided(
            Q.data_ptr(), *Q.stride(), K.data_ptr(), *k_strides, V.data_ptr(), *v_strides, _DTYPE_CODE[self.dtype],
            B, Hq, Hkv, Lq, Lk, D, self.window, self.eps, self.p_round, self.y_round, self.splits,
            self.kernel_size, self.protect_window, self.keep,
            self.scores.data_ptr() if self.scores is not None else None, self.keep_idx.data_ptr(),
            self.k_out.data_ptr(), self.v_out.data_ptr(), self.keep, self.ws.data_ptr(), self.ws.numel(),
            _stream(self.dev))
        _lib.check(rc, "dropkv_evict")
        return self.keep_idx, self.k_out, self.v_out


def decode_workspace(B: int, Hq: int, Hkv: int, D: int, capacity: int, device) -> torch.Tensor:
    """Workspace of ``decode_attention`` for one cache geometry (reusable
    across steps and layers of that geometry)."""
    nbytes = _lib.load().dropkv_decode_workspace_bytes(B, Hq, Hkv, D, capacity)
    if nbytes == 0:
        raise RuntimeError("unsupported decode geometry")
    return _workspace(nbytes, torch.device(device))


def decode_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                     v_cache: torch.Tensor, n_rows: torch.Tensor, scale: float, out: torch.Tensor,
                     workspace: torch.Tensor) -> torch.Tensor:
    """One decode step on preallocated cache buffers (``dropkv_decode_attention``):
    stores k_new / v_new at row ``n_rows`` and writes the attention of q over
    rows 0 .. n_rows into ``out`` [B, 1, Hq, D].  ``n_rows`` (int32, device)
    is not advanced.  Launches only kernels: capturable in a HIP graph."""
    dev = _check_device(q, k_new, v_new, k_cache, v_cache, n_rows, out, workspace)
    if q.dtype not in _DTYPE_CODE or {k_new.dtype, v_new.dtype, k_cache.dtype, v_cache.dtype, out.dtype} != {q.dtype}:
        raise RuntimeError("decode_attention: all tensors must share a bf16/fp16 dtype")
    if n_rows.dtype != torch.int32:
        raise RuntimeError("decode_attention: n_rows must be int32")
    B, Hq, Lq, D = q.shape
    _, Hkv, C, Dk = k_cache.shape
    if Lq != 1 or Dk != D or tuple(k_new.shape) != (B, Hkv, 1, D) or v_new.shape != k_new.shape:
        raise RuntimeError("decode_attention: shape mismatch")
    if k_cache.shape != v_cache.shape or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise RuntimeError("decode_attention: cache buffers must be contiguous and alike")
    if k_new.stride() != v_new.stride():
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    if tuple(out.shape) != (B, 1, Hq, D):
        raise RuntimeError("decode_attention: out must be [B, 1, Hq, D]")
    rc = _lib.load().dropkv_decode_attention(
        q.data_ptr(), q.stride(0), q.stride(1), q.stride(3), k_new.data_ptr(), v_new.data_ptr(),
        k_new.stride(0), k_new.stride(1), k_new.stride(3), k_cache.data_ptr(), v_cache.data_ptr(),
        n_rows.data_ptr(), _DTYPE_CODE[q.dtype], B, Hq, Hkv, D, C, float(scale), out.data_ptr(),
        out.stride(0), out.stride(2), out.stride(3), workspace.data_ptr(), workspace.numel(), _stream(dev))
    _lib.check(rc, "dropkv_decode_attention")
    return out


# The wrappers below check by attribute reads of ~0.1 us each, make outputs like a
# tensor at hand (1.2 us; 1.9 from a shape, 3 for the parts of one) and hand the
# entry point one packed structure: for a call of a few rows their host time is
# the larger part of it.

_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(name: str, index: int, args: bytes) -> None:
    """Entry point ``name`` on the current stream of device ``index``, with that
    device current."""
    fn = getattr(_lib.load(), name)
    if _current_device() == index:
        rc = fn(args, _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream)
    else:
        with torch.cuda.device(index):
            rc = fn(args, torch.cuda.current_stream(index).cuda_stream)
    if rc != 0:
        _lib.check(rc, name)


def _device_index(name: str, *ts) -> int:
    """The device that all of ``ts`` (None left out) are on."""
    index = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != index:
            index = -1
            break
    if index < 0:
        raise RuntimeError(f"{name}: all tensors must be on one ROCm (cuda) device")
    return index


def _differentiating() -> bool:
    """Gradients are recorded, or tangents carried (which no_grad leaves on)."""
    return torch.is_grad_enabled() or _forward_ad._current_level >= 0


def _no_grad(name: str, *ts) -> None:
    backward, forward = torch.is_grad_enabled(), _forward_ad._current_level >= 0
    for t in ts:
        if t is None:
            continue
        if backward and t.requires_grad:
            raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")
        if forward and _forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no gradient: it takes no tensors with a tangent")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with its last axis contiguous."""
    return t if t.stride(-1) == 1 else t.contiguous()


@functools.lru_cache(maxsize=256)
def _tree_bytes(B: int, Hq: int, Hkv: int, D: int, T: int, capacity: int) -> int:
    return _lib.load().dropkv_tree_workspace_bytes(B, Hq, Hkv, D, T, capacity)


def tree_workspace(B: int, Hq: int, Hkv: int, D: int, T: int, capacity: int, device) -> torch.Tensor:
    """Workspace of ``tree_attention`` for one geometry (reusable across steps
    and layers of that geometry, one call at a time)."""
    nbytes = _tree_bytes(B, Hq, Hkv, D, T, capacity)
    if nbytes == 0:
        raise RuntimeError("unsupported tree geometry")
    return _workspace(nbytes, torch.device(device))


_TREE_ARGS = _lib.ARGS["dropkv_tree_attention"].pack


def tree_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor, n_rows: torch.Tensor, scale: float, out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of T drafted tokens per sequence over the cache and over one
    another (``dropkv_tree_attention``): q [B, Hq, T, D], their own rows
    k_new / v_new [B, Hkv, T, D], the buffers [B, Hkv, capacity, D] whose first
    ``n_rows`` rows (int32 on the device, one count or one per sequence) are
    filled.  ``mask`` (bool, [T, T] or [B, T, T]) says which drafted token
    (second to last axis) sees which; without it they are a chain.  Returns
    ``out`` [B, T, Hq, D], which must not lie in an input; a row that sees no key
    is zeros.  Beyond Hq / Hkv * T = 64 the weights may be rounded once to the
    dtype before they meet the values (half a step each; below, 16 bits or
    more).  The buffers are not written: ``tree_commit`` stores the rows of the
    tokens that stand."""
    index = _device_index("tree_attention", q, k_new, v_new, k_cache, v_cache, n_rows, out, workspace, mask)
    if _differentiating():
        _no_grad("tree_attention", q, k_new, v_new, k_cache, v_cache, out)
    dtype = q.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise RuntimeError("tree_attention: the dtype must be bf16 or fp16")
    if not dtype is k_new.dtype is v_new.dtype is k_cache.dtype is v_cache.dtype:
        raise RuntimeError("tree_attention: all tensors must share a dtype")
    shape, kshape, cshape = q.shape, k_new.shape, k_cache.shape
    if len(shape) != 4 or len(kshape) != 4 or v_new.shape != kshape:
        raise RuntimeError("tree_attention: q must be [B, Hq, T, D], k_new and v_new [B, Hkv, T, D]")
    B, Hq, T, D = shape
    if len(cshape) != 4 or v_cache.shape != cshape:
        raise RuntimeError("tree_attention: the cache buffers must be [B, Hkv, capacity, D]")
    cB, Hkv, C, cD = cshape
    if cB != B or cD != D or kshape != (B, Hkv, T, D):
        raise RuntimeError("tree_attention: q, k_new, v_new and the cache buffers do not fit one another")
    k_ptr, v_ptr = k_cache.data_ptr(), v_cache.data_ptr()
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()) or (k_ptr | v_ptr) & 15:
        raise RuntimeError("tree_attention: the cache buffers must be contiguous and 16-byte aligned")
    counts = n_rows.numel()
    if n_rows.dtype is not torch.int32 or (counts != 1 and counts != B) or not n_rows.is_contiguous():
        raise RuntimeError("tree_attention: n_rows must hold one int32 count, or one per sequence")
    m_ptr = m_b = m_t = m_j = 0
    if mask is not None:
        mshape = mask.shape
        if mask.dtype is not torch.bool or (mshape != (T, T) and mshape != (B, T, T)):
            raise RuntimeError("tree_attention: mask must be bool, [T, T] or [B, T, T]")
        m_ptr = mask.data_ptr()
        if len(mshape) == 2:
            m_t, m_j = mask.stride()
        else:
            m_b, m_t, m_j = mask.stride()
    if out is None:
        out = q.new_empty((B, T, Hq, D))
    elif out.shape != (B, T, Hq, D) or out.dtype is not dtype or out.stride(3) != 1:
        raise RuntimeError("tree_attention: out must be [B, T, Hq, D] of q's dtype, D contiguous")
    if not (B and T and Hq):
        return out
    if workspace is None:
        nbytes = _tree_bytes(B, Hq, Hkv, D, T, C)
        if nbytes == 0:
            raise RuntimeError("tree_attention: unsupported geometry")
        workspace = _stream_workspace(nbytes, q.device)
    elif not workspace.is_contiguous():
        raise RuntimeError("tree_attention: the workspace must be contiguous")
    q_b, q_h, q_t, q_d = q.stride()
    if q_d != 1:
        q_b, q_h, q_t, _ = (q := q.contiguous()).stride()
    kn_b, kn_h, kn_t, kn_d = k_new.stride()
    if kn_d != 1:
        kn_b, kn_h, kn_t, _ = (k_new := k_new.contiguous()).stride()
    vn_b, vn_h, vn_t, vn_d = v_new.stride()
    if vn_d != 1:
        vn_b, vn_h, vn_t, _ = (v_new := v_new.contiguous()).stride()
    o_b, o_t, o_h, _ = out.stride()
    _call("dropkv_tree_attention", index, _TREE_ARGS(
        q.data_ptr(), q_b, q_h, q_t, k_new.data_ptr(), kn_b, kn_h, kn_t, v_new.data_ptr(), vn_b, vn_h, vn_t, k_ptr,
        v_ptr, n_rows.data_ptr(), counts > 1, m_ptr, m_b, m_t, m_j, _DTYPE_CODE[dtype], B, Hq, Hkv, T, D, C, scale,
        out.data_ptr(), o_b, o_t, o_h, workspace.data_ptr(), workspace.nbytes))
    return out


_COMMIT_ARGS = _lib.ARGS["dropkv_tree_commit"].pack


def tree_commit(tokens: torch.Tensor, parents: torch.Tensor, choice: torch.Tensor, k_new: torch.Tensor,
                v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, n_rows: torch.Tensor):
    """Which drafted tokens stand, and their rows appended to the caches
    (``dropkv_tree_commit``).  ``tokens`` [B, T] int64 were fed, ``choice``
    [B, T] int64 is the token settled on after each, ``parents`` ([T] or [B, T],
    int32) the trees; node 0 stands, and from a node that stands the walk goes
    to its lowest child whose token is the node's choice.  ``k_new`` / ``v_new``
    [B, H, T, D] and the buffers [B, H, capacity, D], or those of N layers with
    an axis N in front; ``n_rows`` int32, [1] or [B], or [N, 1] or [N, B].
    Returns ``(path [B, T] int32, the nodes that stand, then -1; accepted [B]
    int32)``.  ``n_rows`` is not advanced.  The drafted rows must not lie in the
    buffers themselves."""
    index = _device_index("tree_commit", tokens, parents, choice, k_new, v_new, k_cache, v_cache, n_rows)
    if _differentiating():
        _no_grad("tree_commit", k_new, v_new, k_cache, v_cache)
    tshape = tokens.shape
    if len(tshape) != 2 or choice.shape != tshape or not tokens.dtype is choice.dtype is torch.int64:
        raise RuntimeError("tree_commit: tokens and choice must be int64 [B, T]")
    B, T = tshape
    pshape, cshape = parents.shape, k_cache.shape
    if parents.dtype is not torch.int32 or (pshape != (B, T) and pshape != (T,) and pshape != (1, T)):
        raise RuntimeError("tree_commit: parents must be int32 [T] or [B, T]")
    layers = len(cshape) == 5
    if not (layers or len(cshape) == 4) or v_cache.shape != cshape:
        raise RuntimeError("tree_commit: the buffers must be [B, H, capacity, D] or [N, B, H, capacity, D]")
    *lead, H, C, D = cshape
    if lead[-1] != B or k_new.shape != (*lead, H, T, D) or v_new.shape != k_new.shape:
        raise RuntimeError("tree_commit: tokens, rows and buffers do not fit one another")
    dtype = k_cache.dtype
    if dtype not in _DTYPE_CODE or not dtype is v_cache.dtype is k_new.dtype is v_new.dtype:
        raise RuntimeError("tree_commit: rows and buffers must share a bf16, fp16 or fp32 dtype")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise RuntimeError("tree_commit: the cache buffers must be contiguous")
    N = lead[0] if layers else 1
    nshape = n_rows.shape
    if n_rows.dtype is not torch.int32 or len(nshape) != len(lead) or nshape[-1] not in (1, B) or nshape[0] not in (
            (N,) if layers else (1, B)):
        raise RuntimeError("tree_commit: n_rows must be int32, [1] or [B], or [N, 1] or [N, B]")
    path = torch.empty_like(tokens, dtype=torch.int32, memory_format=torch.contiguous_format)
    accepted = tokens.new_empty((B,), dtype=torch.int32)
    if B == 0:
        return path, accepted
    tokens, choice, parents = tokens.contiguous(), choice.contiguous(), parents.contiguous()
    k_new, v_new = _rows(k_new), _rows(v_new)
    ks, vs, ns = k_new.stride(), v_new.stride(), n_rows.stride()
    if not layers:
        ks, vs, ns = (0, *ks), (0, *vs), (0, *ns)
    _call("dropkv_tree_commit", index, _COMMIT_ARGS(
        tokens.data_ptr(), parents.data_ptr(), T if parents.numel() != T else 0, choice.data_ptr(), path.data_ptr(),
        accepted.data_ptr(), k_new.data_ptr(), *ks[:4], v_new.data_ptr(), *vs[:4], k_cache.data_ptr(),
        v_cache.data_ptr(), n_rows.data_ptr(), ns[0], ns[1] if nshape[-1] > 1 else 0, k_cache.element_size(), N, B, H,
        T, D, C))
    return path, accepted


_ROPE_ARGS = _lib.ARGS["dropkv_norm_rope"].pack


def _rope_out(t, like, name):
    if t is None:
        t = torch.empty_like(like)  # (its layout too, where it is dense)
        if t.stride(3) == 1:
            return t
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if t.shape != like.shape or t.dtype is not like.dtype or t.stride(3) != 1:
        raise RuntimeError(f"norm_rope: {name} must have its input's shape and dtype, D contiguous")
    return t


def norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
              positions: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
              k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, v: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
              v_out: Optional[torch.Tensor] = None):
    """Norms (with ``q_weight`` / ``k_weight`` [D]) and rotation of queries
    [B, Hq, L, D] and keys [B, Hkv, L, D], any strides, in one pass
    (``dropkv_norm_rope``).  ``cos`` and ``sin`` hold the R <= D rotated values'
    factors (value i is paired with i + R/2), in fp32 or q's dtype: each token's
    ([L, R], [1, L, R] or [B, L, R]), or with ``positions`` (int64, [L], [1, L]
    or [B, L]) a table [rows, R]; a position outside the table gives NaN.  With
    ``v`` its rows are copied too.  The outputs may be views of cache buffers
    (``k_buf[:, :, n:n + L]``), or the inputs themselves, and are new tensors
    otherwise.  Returns ``(q_out, k_out)``, or ``(q_out, k_out, v_out)``."""
    index = _device_index("norm_rope", q, k, cos, sin, positions, q_weight, k_weight, v, q_out, k_out, v_out)
    if _differentiating():
        _no_grad("norm_rope", q, k, v, cos, sin, q_weight, k_weight, q_out, k_out, v_out)
    dtype, cdtype = q.dtype, cos.dtype
    if dtype not in _DTYPE_CODE or k.dtype is not dtype or (v is not None and v.dtype is not dtype):
        raise RuntimeError("norm_rope: q, k and v must share a bf16, fp16 or fp32 dtype")
    shape, kshape = q.shape, k.shape
    if len(shape) != 4 or len(kshape) != 4:
        raise RuntimeError("norm_rope: q and k must be [B, H, L, D]")
    B, Hq, L, D = shape
    Hkv = kshape[1]
    if kshape != (B, Hkv, L, D) or (v is not None and v.shape != kshape):
        raise RuntimeError("norm_rope: k and v must be [B, Hkv, L, D]")
    ashape = cos.shape
    if sin.shape != ashape or sin.dtype is not cdtype or (cdtype is not torch.float32 and cdtype is not dtype):
        raise RuntimeError("norm_rope: cos and sin must be alike, fp32 or of q's dtype")
    R = ashape[-1] if ashape else 0
    c_stride = cos.stride()
    if ashape and (c_stride[-1] != 1 or sin.stride() != c_stride):
        cos, sin = cos.contiguous(), sin.contiguous()
        c_stride = cos.stride()
    p_ptr = p_b = c_b = 0
    if positions is not None:
        pshape = positions.shape
        if len(ashape) != 2 or positions.dtype is not torch.int64 or (
                pshape != (B, L) and pshape != (L,) and pshape != (1, L)):
            raise RuntimeError("norm_rope: positions must be int64 [L] or [B, L], with cos and sin [rows, R]")
        positions = positions.contiguous()
        p_ptr, p_b = positions.data_ptr(), L if len(pshape) == 2 and pshape[0] > 1 else 0
    elif ashape == (B, L, R):
        c_b = c_stride[0] if B > 1 else 0
    elif ashape != (L, R) and ashape != (1, L, R):
        raise RuntimeError("norm_rope: cos and sin must be [L, R], [1, L, R] or [B, L, R]")
    qw = kw = w_code = 0
    if q_weight is not None or k_weight is not None:
        weights = [w for w in (q_weight, k_weight) if w is not None]
        wdtype = weights[0].dtype
        for w in weights:
            if w.shape != (D,) or w.dtype is not wdtype or (wdtype is not torch.float32 and wdtype is not dtype):
                raise RuntimeError("norm_rope: norm weights must be [D], fp32 or of q's dtype, and alike")
        w_code = _DTYPE_CODE[wdtype]
        if q_weight is not None:
            q_weight = q_weight.contiguous()
            qw = q_weight.data_ptr()
        if k_weight is not None:
            k_weight = k_weight.contiguous()
            kw = k_weight.data_ptr()
    if v is None and v_out is not None:
        raise RuntimeError("norm_rope: v_out without v")
    q, k = _rows(q), _rows(k)
    q_out, k_out = _rope_out(q_out, q, "q_out"), _rope_out(k_out, k, "k_out")
    v_ptr = v_b = v_h = v_l = vo_ptr = vo_b = vo_h = vo_l = 0
    if v is not None:
        v = _rows(v)
        v_out = _rope_out(v_out, v, "v_out")
        v_ptr, vo_ptr = v.data_ptr(), v_out.data_ptr()
        v_b, v_h, v_l, _ = v.stride()
        vo_b, vo_h, vo_l, _ = v_out.stride()
    if B and L:
        q_b, q_h, q_l, _ = q.stride()
        qo_b, qo_h, qo_l, _ = q_out.stride()
        k_b, k_h, k_l, _ = k.stride()
        ko_b, ko_h, ko_l, _ = k_out.stride()
        _call("dropkv_norm_rope", index, _ROPE_ARGS(
            q.data_ptr(), q_b, q_h, q_l, q_out.data_ptr(), qo_b, qo_h, qo_l, k.data_ptr(), k_b, k_h, k_l,
            k_out.data_ptr(), ko_b, ko_h, ko_l, v_ptr, v_b, v_h, v_l, vo_ptr, vo_b, vo_h, vo_l, qw, kw, w_code,
            cos.data_ptr(), sin.data_ptr(), _DTYPE_CODE[cdtype], c_b, c_stride[-2], p_ptr, p_b, ashape[0],
            _DTYPE_CODE[dtype], B, Hq, Hkv, L, D, R, eps))
    return (q_out, k_out) if v is None else (q_out, k_out, v_out)


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns; the leading axes are the logits'."""

    logprob: Optional[torch.Tensor]  # [...] fp32, None without tokens
    entropy: torch.Tensor            # [...] fp32
    top_logprobs: torch.Tensor       # [..., top] fp32
    top_ids: torch.Tensor            # [..., top] int64


_LOGPROB_ARGS = _lib.ARGS["dropkv_token_logprobs"].pack


@functools.lru_cache(maxsize=256)
def _logprob_bytes(N: int, V: int, top: int) -> int:
    return _lib.load().dropkv_token_logprobs_workspace_bytes(N, V, top)


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """Log probability of a given token, entropy, and the ``top`` (at most 32)
    most probable tokens of every row of ``logits`` [..., V] (bf16, fp16 or
    fp32), in one pass over them (``dropkv_token_logprobs``).  ``tokens`` [...]
    int64: 0 comes out where it is negative, NaN where it is V or more.  The top
    tokens come largest first, the lowest id first among equals."""
    index = _device_index("token_logprobs", logits, tokens)
    if _differentiating():
        _no_grad("token_logprobs", logits)
    dtype, shape, device = logits.dtype, logits.shape, logits.device
    if dtype not in _DTYPE_CODE:
        raise RuntimeError("token_logprobs: logits must be bf16, fp16 or fp32")
    if len(shape) < 1 or shape[-1] < 1:
        raise RuntimeError("token_logprobs: logits must be [..., V]")
    lead, V = shape[:-1], shape[-1]
    if not 0 <= top <= V:
        raise RuntimeError("token_logprobs: top must be in [0, V]")
    if tokens is not None:
        if tokens.dtype is not torch.int64 or tokens.shape != lead:
            raise RuntimeError("token_logprobs: tokens must be int64, of the logits' leading shape")
        tokens = tokens.contiguous()
    x = _rows(logits if len(shape) == 2 else logits.reshape(-1, V))
    N = x.shape[0]
    if tokens is None:
        logprob, entropy = None, logits.new_empty(lead, dtype=torch.float32)
    else:
        logprob = torch.empty_like(tokens, dtype=torch.float32, memory_format=torch.contiguous_format)
        entropy = torch.empty_like(logprob)
    top_lp = logits.new_empty((*lead, top), dtype=torch.float32)
    top_id = torch.empty_like(top_lp, dtype=torch.int64)
    if N:
        nbytes = _logprob_bytes(N, V, top)
        ws = _stream_workspace(nbytes, device) if nbytes else None
        _call("dropkv_token_logprobs", index, _LOGPROB_ARGS(
            x.data_ptr(), x.stride(0), _DTYPE_CODE[dtype], N, V, 0 if tokens is None else tokens.data_ptr(), top,
            0 if logprob is None else logprob.data_ptr(), entropy.data_ptr(), top_lp.data_ptr(), top_id.data_ptr(),
            0 if ws is None else ws.data_ptr(), nbytes))
    return TokenLogprobs(logprob, entropy, top_lp, top_id)


def mfma_selftest(device="cuda") -> torch.Tensor:
    out = torch.empty(16, 16, dtype=torch.float32, device=device)
    rc = _lib.load().dropkv_selftest_mfma(out.data_ptr(), _stream(out.device))
    _lib.check(rc, "dropkv_selftest_mfma")
    return out
