"""Torch-tensor wrappers around the C ABI of libdropkv_amd.so.

PyTorch provides device memory (its caching allocator, also for the
workspaces) and the current HIP stream; all arithmetic runs in the HIP
kernels.  The wrappers check what the kernels assume (device, dtype, layout,
alignment) and raise ``RuntimeError`` otherwise; the reference-compatible
``AssertionError`` guards live in :mod:`dropkv_amd.dropkv_triton`.
"""

from __future__ import annotations

import ctypes
import threading
from typing import NamedTuple, Optional

import torch

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


# One workspace per (device, stream), grown on demand and reused by every
# ``scores`` / ``evict`` call on that stream: calls on one stream run in
# order, so they never use it at the same time.
_shared_ws: dict = {}
_shared_ws_lock = threading.Lock()


def _stream_workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    nbytes = max(int(nbytes), 1)
    if torch.cuda.is_current_stream_capturing():
        return _evict_workspace(nbytes, dev)  # a graph keeps its own (private-pool) workspace
    key = (dev.index, _stream(dev))
    with _shared_ws_lock:
        ws = _shared_ws.get(key)
        if ws is None or ws.numel() < nbytes:
            ws = _evict_workspace(nbytes, dev)
            _shared_ws[key] = ws
    return ws


def release_workspaces() -> None:
    """Drop the per-(device, stream) workspaces kept for calls that bring
    none (they only grow, to the largest call seen on that stream, and are
    otherwise held for the life of the process).  Each goes back to
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


def _call(dev: torch.device, name: str, *args) -> None:
    """Entry point ``name`` on the current stream of ``dev``, with ``dev`` current."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    _lib.check(rc, name)


def _no_grad(name: str, *ts) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with its last axis contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def tree_workspace(B: int, Hq: int, Hkv: int, D: int, T: int, capacity: int, device) -> torch.Tensor:
    """Workspace of ``tree_attention`` for one geometry (reusable across steps
    and layers of that geometry, one call at a time)."""
    nbytes = _lib.load().dropkv_tree_workspace_bytes(B, Hq, Hkv, D, T, capacity)
    if nbytes == 0:
        raise RuntimeError("unsupported tree geometry")
    return _workspace(nbytes, torch.device(device))


def tree_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor, n_rows: torch.Tensor, scale: float, out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of T drafted tokens per sequence over the cache and over one
    another (``dropkv_tree_attention``): q [B, Hq, T, D], their own rows
    k_new / v_new [B, Hkv, T, D], the buffers [B, Hkv, capacity, D] whose first
    ``n_rows`` rows (int32 on the device, one count or one per sequence) are
    filled.  ``mask`` (bool, [T, T] or [B, T, T]) says which drafted token
    (second to last axis) sees which; without it they are a chain.  Returns
    ``out`` [B, T, Hq, D]; a row that sees no key is zeros.  The buffers are not
    written: ``tree_commit`` stores the rows of the tokens that stand."""
    dev = _check_device(q, k_new, v_new, k_cache, v_cache, n_rows)
    _no_grad("tree_attention", q, k_new, v_new, k_cache, v_cache)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError("tree_attention: the dtype must be bf16 or fp16")
    for t in (k_new, v_new, k_cache, v_cache):
        if t.dtype != q.dtype:
            raise RuntimeError("tree_attention: all tensors must share a dtype")
    if q.dim() != 4 or k_new.dim() != 4:
        raise RuntimeError("tree_attention: q, k_new and v_new must be [B, H, T, D]")
    B, Hq, T, D = q.shape
    _check_buffer(k_cache, "k_cache")
    _check_buffer(v_cache, "v_cache")
    Hkv, C = k_cache.shape[1], k_cache.shape[2]
    if k_new.shape != (B, Hkv, T, D) or v_new.shape != k_new.shape:
        raise RuntimeError("tree_attention: k_new and v_new must be [B, Hkv, T, D]")
    if k_cache.shape != (B, Hkv, C, D) or v_cache.shape != k_cache.shape:
        raise RuntimeError("tree_attention: the cache buffers must be [B, Hkv, capacity, D]")
    if n_rows.dtype != torch.int32 or n_rows.numel() not in (1, B) or not n_rows.is_contiguous():
        raise RuntimeError("tree_attention: n_rows must hold one int32 count, or one per sequence")
    m_ptr, m_strides = None, (0, 0, 0)
    if mask is not None:
        _check_device(q, mask)
        if mask.dtype != torch.bool or mask.shape not in ((T, T), (B, T, T)):
            raise RuntimeError("tree_attention: mask must be bool, [T, T] or [B, T, T]")
        m_ptr = mask.data_ptr()
        m_strides = (0, *mask.stride()) if mask.dim() == 2 else mask.stride()
    if out is None:
        out = torch.empty(B, T, Hq, D, dtype=q.dtype, device=dev)
    else:
        _check_device(q, out)
        if out.shape != (B, T, Hq, D) or out.dtype != q.dtype or (out.stride(3) != 1 and D > 1):
            raise RuntimeError("tree_attention: out must be [B, T, Hq, D] of q's dtype, D contiguous")
    if workspace is None:
        workspace = tree_workspace(B, Hq, Hkv, D, T, C, dev)
    else:
        _check_device(q, workspace)
    q, k_new, v_new = _rows(q), _rows(k_new), _rows(v_new)
    qs, ks, vs, os = q.stride(), k_new.stride(), v_new.stride(), out.stride()
    _call(dev, "dropkv_tree_attention", q.data_ptr(), qs[0], qs[1], qs[2], k_new.data_ptr(), ks[0], ks[1], ks[2],
          v_new.data_ptr(), vs[0], vs[1], vs[2], k_cache.data_ptr(), v_cache.data_ptr(), n_rows.data_ptr(),
          int(n_rows.numel() > 1), m_ptr, *m_strides, _DTYPE_CODE[q.dtype], B, Hq, Hkv, T, D, C, float(scale),
          out.data_ptr(), os[0], os[1], os[2], workspace.data_ptr(), workspace.numel() * workspace.element_size())
    return out


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
    int32)``.  ``n_rows`` is not advanced."""
    dev = _check_device(tokens, parents, choice, k_new, v_new, k_cache, v_cache, n_rows)
    _no_grad("tree_commit", k_new, v_new, k_cache, v_cache)
    if tokens.dim() != 2 or choice.shape != tokens.shape or tokens.dtype != torch.int64 or choice.dtype != torch.int64:
        raise RuntimeError("tree_commit: tokens and choice must be int64 [B, T]")
    B, T = tokens.shape
    if parents.dtype != torch.int32 or parents.shape not in ((T,), (1, T), (B, T)):
        raise RuntimeError("tree_commit: parents must be int32 [T] or [B, T]")
    if k_cache.dim() not in (4, 5) or k_new.dim() != k_cache.dim():
        raise RuntimeError("tree_commit: rows and buffers must be [B, H, ., D] or [N, B, H, ., D]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise RuntimeError("tree_commit: the cache buffers must be contiguous")
    *lead, H, C, D = k_cache.shape
    if lead[-1] != B or k_new.shape != (*lead, H, T, D) or v_new.shape != k_new.shape or v_cache.shape != k_cache.shape:
        raise RuntimeError("tree_commit: shape mismatch")
    if not k_cache.dtype == v_cache.dtype == k_new.dtype == v_new.dtype or k_cache.dtype not in _DTYPE_CODE:
        raise RuntimeError("tree_commit: rows and buffers must share a bf16, fp16 or fp32 dtype")
    if n_rows.dtype != torch.int32 or n_rows.dim() != len(lead) or any(
            a not in (1, b) for a, b in zip(n_rows.shape, lead)) or (len(lead) == 2 and n_rows.shape[0] != lead[0]):
        raise RuntimeError("tree_commit: n_rows must be int32, [1] or [B], or [N, 1] or [N, B]")
    N = lead[0] if len(lead) == 2 else 1
    path = torch.empty(B, T, dtype=torch.int32, device=dev)
    accepted = torch.empty(B, dtype=torch.int32, device=dev)
    if path.numel() == 0:
        return path, accepted
    tokens, choice, parents = tokens.contiguous(), choice.contiguous(), parents.contiguous()
    k_new, v_new = _rows(k_new), _rows(v_new)
    ks, vs, ns = k_new.stride()[:-1], v_new.stride()[:-1], n_rows.expand(lead).stride()
    if N == 1 and len(lead) == 1:
        ks, vs, ns = (0, *ks), (0, *vs), (0, *ns)
    _call(dev, "dropkv_tree_commit", tokens.data_ptr(), parents.data_ptr(), T if parents.numel() > T else 0,
          choice.data_ptr(), path.data_ptr(), accepted.data_ptr(), k_new.data_ptr(), *ks, v_new.data_ptr(), *vs,
          k_cache.data_ptr(), v_cache.data_ptr(), n_rows.data_ptr(), *ns, k_cache.element_size(), N, B, H, T, D, C)
    return path, accepted


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
    dev = _check_device(q, k, cos, sin)
    _no_grad("norm_rope", q, k, v, cos, sin, q_weight, k_weight)
    if q.dtype not in _DTYPE_CODE or k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        raise RuntimeError("norm_rope: q, k and v must share a bf16, fp16 or fp32 dtype")
    if q.dim() != 4 or k.dim() != 4:
        raise RuntimeError("norm_rope: q and k must be [B, H, L, D]")
    B, Hq, L, D = q.shape
    Hkv = k.shape[1]
    if k.shape != (B, Hkv, L, D) or (v is not None and v.shape != k.shape):
        raise RuntimeError("norm_rope: k and v must be [B, Hkv, L, D]")
    R = cos.shape[-1]
    if sin.shape != cos.shape or sin.dtype != cos.dtype or cos.dtype not in (torch.float32, q.dtype):
        raise RuntimeError("norm_rope: cos and sin must be alike, fp32 or of q's dtype")
    p_ptr, p_sb = None, 0
    if positions is not None:
        _check_device(q, positions)
        if cos.dim() != 2 or positions.dtype != torch.int64 or positions.shape not in ((L,), (1, L), (B, L)):
            raise RuntimeError("norm_rope: positions must be int64 [L] or [B, L], with cos and sin [rows, R]")
        positions = positions.contiguous()
        p_ptr, p_sb = positions.data_ptr(), L if positions.numel() > L else 0
    elif cos.shape not in ((L, R), (1, L, R), (B, L, R)):
        raise RuntimeError("norm_rope: cos and sin must be [L, R], [1, L, R] or [B, L, R]")
    if cos.stride(-1) != 1 or sin.stride() != cos.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    c_sb = cos.stride(0) if positions is None and cos.dim() == 3 and cos.shape[0] > 1 else 0
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        _check_device(q, w)
        if w.shape != (D,) or w.dtype not in (torch.float32, q.dtype) or w.dtype != weights[0].dtype:
            raise RuntimeError("norm_rope: norm weights must be [D], fp32 or of q's dtype, and alike")
    q_weight, k_weight = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    if v is None and v_out is not None:
        raise RuntimeError("norm_rope: v_out without v")

    def target(t, like, name):
        if t is None:
            return torch.empty(like.shape, dtype=q.dtype, device=dev)
        _check_device(q, t)
        if t.shape != like.shape or t.dtype != q.dtype or t.stride(3) != 1:
            raise RuntimeError(f"norm_rope: {name} must have its input's shape and dtype, D contiguous")
        return t

    q_out, k_out = target(q_out, q, "q_out"), target(k_out, k, "k_out")
    outs = (q_out, k_out)
    q, k = _rows(q), _rows(k)
    pairs = [(q, q_out), (k, k_out)]
    if v is not None:
        v_out = target(v_out, v, "v_out")
        v = _rows(v)
        outs += (v_out,)
        pairs.append((v, v_out))
    if q.numel() == 0:
        return outs
    strides = (ctypes.c_int64 * 18)(*[s for pair in pairs for t in pair for s in t.stride()[:3]])
    args = []
    for i, pair in enumerate(pairs):
        for j, t in enumerate(pair):
            args += [t.data_ptr(), ctypes.addressof(strides) + 24 * (2 * i + j)]
    if v is None:
        args += [None] * 4
    _call(dev, "dropkv_norm_rope", *args, None if q_weight is None else q_weight.data_ptr(),
          None if k_weight is None else k_weight.data_ptr(), _DTYPE_CODE[weights[0].dtype] if weights else 0,
          cos.data_ptr(), sin.data_ptr(), _DTYPE_CODE[cos.dtype], c_sb, cos.stride(-2), p_ptr, p_sb, cos.shape[0],
          _DTYPE_CODE[q.dtype], B, Hq, Hkv, L, D, R, float(eps))
    return outs


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns; the leading axes are the logits'."""

    logprob: Optional[torch.Tensor]  # [...] fp32, None without tokens
    entropy: torch.Tensor            # [...] fp32
    top_logprobs: torch.Tensor       # [..., top] fp32
    top_ids: torch.Tensor            # [..., top] int64


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """Log probability of a given token, entropy, and the ``top`` (at most 32)
    most probable tokens of every row of ``logits`` [..., V] (bf16, fp16 or
    fp32), in one pass over them (``dropkv_token_logprobs``).  ``tokens`` [...]
    int64: 0 comes out where it is negative, NaN where it is V or more.  The top
    tokens come largest first, the lowest id first among equals."""
    dev = _check_device(logits)
    _no_grad("token_logprobs", logits)
    if logits.dtype not in _DTYPE_CODE:
        raise RuntimeError("token_logprobs: logits must be bf16, fp16 or fp32")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError("token_logprobs: logits must be [..., V]")
    *lead, V = logits.shape
    if not 0 <= top <= V:
        raise RuntimeError("token_logprobs: top must be in [0, V]")
    if tokens is not None:
        _check_device(logits, tokens)
        if tokens.dtype != torch.int64 or list(tokens.shape) != lead:
            raise RuntimeError("token_logprobs: tokens must be int64, of the logits' leading shape")
        tokens = tokens.contiguous()
    x = _rows(logits.reshape(-1, V))
    N = x.shape[0]
    logprob = None if tokens is None else torch.empty(lead, dtype=torch.float32, device=dev)
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    top_lp = torch.empty(*lead, top, dtype=torch.float32, device=dev)
    top_id = torch.empty(*lead, top, dtype=torch.int64, device=dev)
    res = TokenLogprobs(logprob, entropy, top_lp, top_id)
    if N == 0:
        return res
    nbytes = _lib.load().dropkv_token_logprobs_workspace_bytes(N, V, top)
    ws = _workspace(nbytes, dev) if nbytes else None
    _call(dev, "dropkv_token_logprobs", x.data_ptr(), x.stride(0), _DTYPE_CODE[x.dtype], N, V,
          None if tokens is None else tokens.data_ptr(), int(top), None if logprob is None else logprob.data_ptr(),
          entropy.data_ptr(), top_lp.data_ptr(), top_id.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    return res


def mfma_selftest(device="cuda") -> torch.Tensor:
    out = torch.empty(16, 16, dtype=torch.float32, device=device)
    rc = _lib.load().dropkv_selftest_mfma(out.data_ptr(), _stream(out.device))
    _lib.check(rc, "dropkv_selftest_mfma")
    return out
