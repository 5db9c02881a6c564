"""Drop-in attention entry points backed by the gfx950 HIP kernels in libwdrz_attn.so.

Two functions mirror the reference's two attention seams, with the same names, argument
meaning and output layout:

* :func:`flash_attn_with_kvcache` — the cached decoder path. Same signature as the dispatcher
  at reference ``src/whisperdrz/model.py:88-95`` and the semantics of its torch fallback
  ``_sdpa_attn_with_kvcache`` (``model.py:20-76``): in-place K/V append at ``cache_seqlens``,
  bottom-right causal mask over the slot, ``cache_batch_idx`` slot mapping; cross-attention
  (``k is None``) reads every cache row.
* :func:`scaled_dot_product_attention` — the dense path used by
  ``MultiHeadAttention.qkv_attention`` (``model.py:276-298``, the SDPA call at 288-296), for the
  encoder (non-causal, L=1500) and the uncached decoder (top-left causal).

There is deliberately no CPU or torch fallback here: CPU tensors, unsupported shapes and a
missing library raise. The reference keeps its own fallback for CPU tensors (its dispatcher
only routes ``q.is_cuda`` calls to the accelerated implementation).
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch

from . import _lib

__all__ = [
    "flash_attn_with_kvcache",
    "flash_attn_with_kvcache8",
    "scaled_dot_product_attention",
    "qkv_attention",
    "flash_attn_with_kvpages",
    "packed_attention",
    "kvcache_workspace_size",
    "kvcache8_workspace_size",
    "kvpages_workspace_size",
    "WorkspaceCache",
]

_DTYPES = {torch.float32: _lib.WDRZ_F32, torch.float16: _lib.WDRZ_F16, torch.bfloat16: _lib.WDRZ_BF16}
_DTYPES16 = {torch.float16: _lib.WDRZ_F16, torch.bfloat16: _lib.WDRZ_BF16}
HEAD_DIM = 64


def _dtype_code(t: torch.Tensor, name: str) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{name}: dtype {t.dtype} is not supported (float32, float16, bfloat16)") from None


def _check_cuda(name: str, t: torch.Tensor, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(
            f"{name} is on {t.device}: whisperdrz_amd runs on the GPU only (the reference keeps "
            "its torch fallback for CPU tensors)"
        )
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")


def _stream_handle() -> int:
    return torch.cuda.current_stream().cuda_stream


# The handle of a device's current stream and the current device's index. The public calls build a Stream
# object and look at the initialisation each time: 1 us of a 7 us call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _raise(rc: int, what: str) -> None:
    msg = _lib.last_error()
    if rc == _lib.WDRZ_EUNSUPPORTED:
        raise NotImplementedError(f"{what}: {msg}")
    if rc == _lib.WDRZ_EINVAL or rc == _lib.WDRZ_EWORKSPACE:
        raise ValueError(f"{what}: {msg}")
    raise RuntimeError(f"{what}: {msg}")


class WorkspaceCache:
    """Per-(device, stream) split-KV workspace, grown on demand and then reused.

    The workspace holds per-row arrival counters that must be zero before a call; every call
    leaves them zero again, so a buffer is zero-filled once, when it is allocated. Calls on
    one stream are ordered, so they can share a buffer; calls on different streams (e.g. the
    reference's side ``prefill_stream``) get different buffers. Call :meth:`reserve` before
    capturing a hipGraph so no allocation happens inside capture.
    """

    def __init__(self) -> None:
        self._bufs: dict[tuple[int, int], torch.Tensor] = {}

    def get(self, device: torch.device, nbytes: int) -> Optional[torch.Tensor]:
        if nbytes <= 0:
            return None
        key = (device.index if device.index is not None else torch.cuda.current_device(), _stream_handle())
        buf = self._bufs.get(key)
        if buf is None or buf.numel() < nbytes:
            buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            self._bufs[key] = buf
        return buf

    def reserve(self, device: torch.device, nbytes: int) -> None:
        self.get(device, nbytes)

    def clear(self) -> None:
        self._bufs.clear()


_WORKSPACES = WorkspaceCache()


def kvcache_workspace_size(batch: int, sq: int, n_heads: int, head_dim: int, max_seq: int) -> int:
    """Bytes of split-KV workspace :func:`flash_attn_with_kvcache` needs for these sizes."""
    return int(_lib.load().wdrz_attn_kvcache_workspace_size(batch, sq, n_heads, head_dim, max_seq))


def _as_int32(name: str, t, B: int, device: torch.device) -> torch.Tensor:
    if isinstance(t, int):
        return torch.full((B,), t, dtype=torch.int32, device=device)
    _check_cuda(name, t, device)
    if t.dim() != 1 or t.shape[0] != B:
        raise ValueError(f"{name} must have shape [{B}], got {tuple(t.shape)}")
    if t.dtype != torch.int32:
        if t.dtype not in (torch.int64, torch.int16, torch.uint8, torch.int8):
            raise TypeError(f"{name} must be an integer tensor, got {t.dtype}")
        t = t.to(torch.int32)
    if t.stride(0) != 1:
        t = t.contiguous()
    return t


def flash_attn_with_kvcache(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    cache_seqlens=None,
    cache_batch_idx: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    *,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of ``q`` against a slot KV cache (reference ``model.py:20-95``).

    ``out`` and ``workspace`` are keyword-only extensions: a preallocated output, and a
    caller-owned split-KV workspace (zero-filled before its first use; see
    :func:`kvcache_workspace_size`). Without ``workspace`` a per-stream cached one is used.

    Shapes: ``q`` ``[B, sq, H, D]``; ``k_cache``/``v_cache`` ``[n_slots, Lmax, H, D]`` (any
    strides with a contiguous last dim, e.g. head-major storage viewed as slot-major);
    ``k``/``v`` ``[B, sq, H, D]``; ``cache_seqlens`` int32 ``[B]`` (pre-append lengths);
    ``cache_batch_idx`` int32 ``[B]`` batch row -> slot. Returns ``[B, sq, H, D]`` in q's dtype.

    With ``k``/``v`` given they are written in place at rows ``cache_seqlens[b] + t`` of slot
    ``cache_batch_idx[b]`` and query ``t`` attends keys ``j <= cache_seqlens[b] + t``; the
    lengths themselves are not modified (the caller bumps them, ``model.py:602-607``). Without
    them the attention is non-causal over all ``Lmax`` rows. As in the reference fallback the
    mask follows from whether ``k`` is given; ``causal`` is accepted for signature parity.
    """
    lib = _lib.load()
    device = q.device
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)):
        _check_cuda(name, t, device)
    if q.dim() != 4 or k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("q, k_cache and v_cache must be 4-D ([B, sq, H, D] / [n_slots, Lmax, H, D])")
    B, sq, H, D = q.shape
    S, Lmax, Hc, Dc = k_cache.shape
    if tuple(v_cache.shape) != (S, Lmax, Hc, Dc):
        raise ValueError(f"v_cache shape {tuple(v_cache.shape)} != k_cache shape {tuple(k_cache.shape)}")
    if (Hc, Dc) != (H, D):
        raise ValueError(f"cache heads/head_dim {(Hc, Dc)} do not match q {(H, D)}")
    dt = _dtype_code(q, "q")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise TypeError("k_cache and v_cache must have q's dtype")
    has_new = k is not None or v is not None
    if has_new:
        if k is None or v is None:
            raise ValueError("k and v must be given together")
        _check_cuda("k", k, device)
        _check_cuda("v", v, device)
        if tuple(k.shape) != (B, sq, H, D) or tuple(v.shape) != (B, sq, H, D):
            raise ValueError(f"k/v must have shape {(B, sq, H, D)}")
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise TypeError("k and v must have q's dtype")
        if cache_seqlens is None:
            raise ValueError("cache_seqlens is required when k/v are given")
        seqlens = _as_int32("cache_seqlens", cache_seqlens, B, device)
    else:
        seqlens = None
    bidx = None if cache_batch_idx is None else _as_int32("cache_batch_idx", cache_batch_idx, B, device)
    if _lib.debug_mode():  # host copies of the metadata: debugging runs only, not graph capture
        from .debug import check_kvcache_metadata

        check_kvcache_metadata(seqlens.cpu().numpy() if seqlens is not None else None,
                               bidx.cpu().numpy() if bidx is not None else None, sq, S, Lmax, has_new)
    if softmax_scale is None:
        softmax_scale = D ** -0.5
    if out is None:
        out = torch.empty((B, sq, H, D), dtype=q.dtype, device=device)
    else:
        _check_cuda("out", out, device)
        if tuple(out.shape) != (B, sq, H, D) or out.dtype != q.dtype:
            raise ValueError("out must match q's shape and dtype")
    if B == 0 or sq == 0:
        return out
    nbytes = int(lib.wdrz_attn_kvcache_workspace_size(B, sq, H, D, Lmax))
    if nbytes > 0:
        if workspace is None:
            workspace = _WORKSPACES.get(device, nbytes)
        elif workspace.numel() * workspace.element_size() < nbytes:
            raise ValueError(f"workspace too small: need {nbytes} bytes")
    ws_ptr = workspace.data_ptr() if (nbytes > 0 and workspace is not None) else None
    ws_bytes = workspace.numel() * workspace.element_size() if ws_ptr else 0
    rc = lib.wdrz_attn_kvcache(
        dt,
        q.data_ptr(),
        k_cache.data_ptr(),
        v_cache.data_ptr(),
        k.data_ptr() if has_new else None,
        v.data_ptr() if has_new else None,
        seqlens.data_ptr() if seqlens is not None else None,
        bidx.data_ptr() if bidx is not None else None,
        out.data_ptr(),
        B, sq, H, D, S, Lmax,
        _lib.strides4(q.stride()),
        _lib.strides4(k_cache.stride()),
        _lib.strides4(v_cache.stride()),
        _lib.strides4(k.stride() if has_new else (0, 0, 0, 1)),
        _lib.strides4(v.stride() if has_new else (0, 0, 0, 1)),
        _lib.strides4(out.stride()),
        float(softmax_scale),
        int(bool(causal)),
        ws_ptr,
        ws_bytes,
        _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "flash_attn_with_kvcache")
    return out


def _check_ids(name: str, t: torch.Tensor, B: int, device: torch.device) -> torch.Tensor:
    """An int32 [B] tensor on ``device`` as it is, anything else as :func:`_as_int32` takes it."""
    if isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.device == device and t.shape == (B,) and t.is_contiguous():
        return t
    return _as_int32(name, t, B, device)


@functools.lru_cache(maxsize=1024)
def kvcache8_workspace_size(batch: int, sq: int, n_heads: int, max_seq: int) -> int:
    """Bytes of split-KV workspace :func:`flash_attn_with_kvcache8` needs for these sizes."""
    return int(_lib.load().wdrz_attn_kvcache8_workspace_size(batch, sq, n_heads, max_seq))


def flash_attn_with_kvcache8(
    q: torch.Tensor,
    cache,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    cache_seqlens=None,
    cache_batch_idx: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    *,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """:func:`flash_attn_with_kvcache` against a slot cache held in 8 bits (a ``FlashKVCache8``).

    ``q`` ``[B, sq, H, 64]`` in bf16 or fp16; ``cache_batch_idx`` ``[B]`` row -> slot (identity if None).

    With ``k`` / ``v`` ``[B, sq, H, 64]`` (a cache with a ring): they are appended at ``cache_seqlens[b]`` of
    the row's slot and query ``t`` attends positions ``j <= cache_seqlens[b] + t``: those below the last
    multiple of 32 as the codes' values, the newer ones as they came. The lengths are not modified. Rows
    that name one slot must name one length; the last row's ``k`` / ``v`` then count for all of them (rows
    that disagree give NaN and append nothing; ``WDRZ_DEBUG=1`` raises).
    Without them every query attends the first ``cache_seqlens[b]`` positions of the slot, by default all
    of them (a cache with a ring needs the lengths); a row of no positions gives zeros.
    A slot or length out of range gives NaN rows and writes nothing.

    ``out`` is a preallocated output, ``workspace`` a caller-owned split-KV workspace (zero-filled before
    its first use; :func:`kvcache8_workspace_size`). Without it calls of one stream share a cached one, and
    a call that is captured into a graph gets its own, cleared by every replay.
    """
    if not (isinstance(q, torch.Tensor) and q.is_cuda):
        _check_cuda("q", q, q.device if isinstance(q, torch.Tensor) else None)
    device, shape, dtype = q.device, q.shape, q.dtype
    if cache.device != device:
        raise RuntimeError(f"the cache is on {cache.device}, expected {device}")
    if len(shape) != 4:
        raise ValueError("q must be 4-D ([B, sq, H, 64])")
    B, sq, H, D = shape
    if H != cache.n_heads or D != cache.head_dim:
        raise ValueError(f"cache heads/head_dim {(cache.n_heads, cache.head_dim)} do not match q {(H, D)}")
    dt = _DTYPES16.get(dtype)
    if dt is None:
        raise TypeError(f"q: dtype {dtype} is not supported (bfloat16, float16)")
    if cache.has_ring and dtype != cache.dtype:
        raise TypeError(f"q must have the cache's dtype {cache.dtype}")
    k_ptr = k_strides = v_ptr = v_strides = len_ptr = idx_ptr = ws_ptr = None
    if k is not None or v is not None:
        if k is None or v is None:
            raise ValueError("k and v must be given together")
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor) or t.device != device:
                _check_cuda(name, t, device)
            if t.shape != shape:
                raise ValueError(f"{name} must have shape {(B, sq, H, D)}")
            if t.dtype is not dtype:
                raise TypeError("k and v must have q's dtype")
        if not cache.has_ring:
            raise ValueError("appending needs a cache with a ring")
        k_ptr, k_strides, v_ptr, v_strides = k.data_ptr(), _lib.strides(k.stride()), v.data_ptr(), _lib.strides(v.stride())
    if cache_seqlens is not None:
        cache_seqlens = _check_ids("cache_seqlens", cache_seqlens, B, device)
        len_ptr = cache_seqlens.data_ptr()
    elif cache.has_ring:
        raise ValueError("cache_seqlens is required when k/v are given and for a cache with a ring")
    if cache_batch_idx is not None:
        cache_batch_idx = _check_ids("cache_batch_idx", cache_batch_idx, B, device)
        idx_ptr = cache_batch_idx.data_ptr()
    if out is None:  # like a contiguous q: 1.2 us on the host, empty 2.2
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(shape, dtype=dtype, device=device)
    else:
        _check_cuda("out", out, device)
        if out.shape != shape or out.dtype != dtype:
            raise ValueError("out must match q's shape and dtype")
    if B == 0 or sq == 0:
        return out
    index = device.index
    if index != _current_device():  # launches go to the current device
        with torch.cuda.device(index):
            return flash_attn_with_kvcache8(q, cache, k, v, cache_seqlens, cache_batch_idx, softmax_scale, out=out,
                                            workspace=workspace)
    lib, ws_bytes = _lib.load(), 0
    nbytes = kvcache8_workspace_size(B, sq, H, cache.max_seq_length)
    if nbytes:
        if workspace is None:
            # a captured call's own: another graph captured on this stream may be replayed beside its graph
            workspace = (torch.zeros(nbytes, dtype=torch.uint8, device=device)
                         if torch.cuda.is_current_stream_capturing() else _WORKSPACES.get(device, nbytes))
        else:
            _check_cuda("workspace", workspace, device)
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if ws_bytes < nbytes:
            raise ValueError(f"workspace too small: need {nbytes} bytes")
    rc = lib.wdrz_attn_kvcache8(
        dt, cache.struct, q.data_ptr(), _lib.strides(q.stride()), k_ptr, k_strides, v_ptr, v_strides, len_ptr, idx_ptr,
        out.data_ptr(), _lib.strides(out.stride()), B, sq, 0.125 if softmax_scale is None else softmax_scale, ws_ptr,
        ws_bytes, _raw_stream(index),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "flash_attn_with_kvcache8")
    return out


@functools.lru_cache(maxsize=1024)
def kvpages_workspace_size(batch: int, sq: int, n_heads: int, n_kv_heads: int, head_dim: int, max_seq: int) -> int:
    """Bytes of split-KV workspace :func:`flash_attn_with_kvpages` needs for these sizes."""
    return int(_lib.load().wdrz_attn_kvpages_workspace_size(batch, sq, n_heads, n_kv_heads, head_dim, max_seq))


# Workspaces by (device, stream) whose counters stand at their start, apart from _WORKSPACES: calls of other shapes leave
# the counters where they are, so nothing but they has to be zero after a call.
_COUNTED_WORKSPACES: dict[tuple[int, int], torch.Tensor] = {}
_COUNTER_BYTES = 4096 * 4


def _counted_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """The current stream's workspace of ``device``, the current device; a captured call gets its own, its counters cleared by
    every replay (another graph captured on this stream may be replayed beside its graph)."""
    if torch.cuda.is_current_stream_capturing():
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        buf[:_COUNTER_BYTES].zero_()
        return buf
    key = (device.index, _raw_stream(device.index))
    buf = _COUNTED_WORKSPACES.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = _COUNTED_WORKSPACES[key] = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
    return buf


def flash_attn_with_kvpages(
    q: torch.Tensor,
    cache,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    cache_seqlens=None,
    cache_batch_idx: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    *,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """:func:`flash_attn_with_kvcache` against a paged cache (a ``FlashKVPages``), with grouped heads.

    ``q`` ``[B, sq, H, D]`` in the cache's dtype, H a multiple of the cache's heads (query head h reads head
    ``h // (H / n_heads)``); ``cache_seqlens`` ``[B]`` (a plan's ``starts``); ``cache_batch_idx`` ``[B]`` row -> stream
    (identity if None). The streams' own ``seq_lens`` are not read.

    With ``k`` / ``v`` ``[B, sq, n_heads, D]``: they are written at positions ``cache_seqlens[b] + t``, whose pages
    ``PageTables.plan`` has given, and query ``t`` attends positions ``j <= cache_seqlens[b] + t``. Without them every
    query attends the first ``cache_seqlens[b]`` positions; a row of none gives zeros.
    A stream or length out of range (a start of -1 among them) gives NaN rows and writes nothing; so do rows that
    append to one stream in one call. A page out of range gives NaN too (``WDRZ_DEBUG=1`` raises for all of these).

    ``out`` is a preallocated output, ``workspace`` a caller-owned split-KV workspace (zero-filled before its first
    use; :func:`kvpages_workspace_size`). Without it calls of one stream share a cached one, and a call that is
    captured into a graph gets its own, cleared by every replay.
    """
    if not (isinstance(q, torch.Tensor) and q.is_cuda):
        _check_cuda("q", q, q.device if isinstance(q, torch.Tensor) else None)
    device, shape, dtype = q.device, q.shape, q.dtype
    if cache.device != device:
        raise RuntimeError(f"the cache is on {cache.device}, expected {device}")
    if len(shape) != 4:
        raise ValueError("q must be 4-D ([B, sq, H, D])")
    B, sq, H, D = shape
    heads = cache.n_heads
    if H % heads or H == 0 or D != cache.head_dim:
        raise ValueError(f"cache heads/head_dim {(heads, cache.head_dim)} do not match q {(H, D)}")
    if dtype != cache.dtype:
        raise TypeError(f"q must have the cache's dtype {cache.dtype}")
    k_ptr = k_strides = v_ptr = v_strides = idx_ptr = ws_ptr = None
    if k is not None or v is not None:
        if k is None or v is None:
            raise ValueError("k and v must be given together")
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor) or t.device != device:
                _check_cuda(name, t, device)
            if t.shape != (B, sq, heads, D):
                raise ValueError(f"{name} must have shape {(B, sq, heads, D)}")
            if t.dtype is not dtype:
                raise TypeError("k and v must have q's dtype")
        k_ptr, k_strides, v_ptr, v_strides = k.data_ptr(), _lib.strides(k.stride()), v.data_ptr(), _lib.strides(v.stride())
    if cache_seqlens is None:
        raise ValueError("cache_seqlens is required")
    cache_seqlens = _check_ids("cache_seqlens", cache_seqlens, B, device)
    if cache_batch_idx is not None:
        cache_batch_idx = _check_ids("cache_batch_idx", cache_batch_idx, B, device)
        idx_ptr = cache_batch_idx.data_ptr()
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(B, sq, H, D, dtype=dtype, device=device)
    else:
        _check_cuda("out", out, device)
        if out.shape != shape or out.dtype != dtype:
            raise ValueError("out must match q's shape and dtype")
    if B == 0 or sq == 0:
        return out
    index = device.index
    if index != _current_device():  # launches go to the current device
        with torch.cuda.device(index):
            return flash_attn_with_kvpages(q, cache, k, v, cache_seqlens, cache_batch_idx, softmax_scale, out=out,
                                           workspace=workspace)
    lib, ws_bytes = _lib.load(), 0
    nbytes = kvpages_workspace_size(B, sq, H, heads, D, cache.max_seq_length)
    if nbytes:
        if workspace is None:
            workspace = _counted_workspace(device, nbytes)
        else:
            _check_cuda("workspace", workspace, device)
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if ws_bytes < nbytes:
            raise ValueError(f"workspace too small: need {nbytes} bytes")
    rc = lib.wdrz_attn_kvpages(
        _DTYPES16[dtype], cache.struct, cache.page_tables.struct, q.data_ptr(), _lib.strides(q.stride()), k_ptr, k_strides,
        v_ptr, v_strides, cache_seqlens.data_ptr(), idx_ptr, out.data_ptr(), _lib.strides(out.stride()), B, sq, H,
        D ** -0.5 if softmax_scale is None else softmax_scale, ws_ptr, ws_bytes, _raw_stream(index),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "flash_attn_with_kvpages")
    return out


def packed_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    cu_seqlens_k: Optional[torch.Tensor] = None,
    causal: bool = True,
    scale: Optional[float] = None,
    *,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of sequences of different lengths, packed without padding: ``q`` ``[T, H, D]``, ``k`` and ``v``
    ``[Tk, Hk, D]`` in bf16 or fp16, D 64 or 128, H a multiple of Hk (query head h reads head ``h // (H / Hk)``); strided
    views of a projection where the last dimension is contiguous.

    Sequence i is rows ``cu_seqlens[i] .. cu_seqlens[i + 1] - 1`` of the queries (int32 ``[B + 1]``, ascending; a
    plan's ``cu_seqlens``) and, with ``cu_seqlens_k``, rows of the keys of its own. ``causal``: query t sees the keys
    ``j <= t + (keys - queries)`` of its sequence, the last query all of them; else every query sees all. A query that
    sees none gives zeros. Rows that no sequence holds are left as they are in ``out`` (a new one is not filled there).
    Scores, softmax and sums are fp32; a probability is rounded once to q's type before it weighs a value (half a step, 2^-8 or 2^-11
    of it), where :func:`flash_attn_with_kvpages` keeps what the rounding leaves. Inference only.
    """
    if not (isinstance(q, torch.Tensor) and q.is_cuda):
        _check_cuda("q", q, q.device if isinstance(q, torch.Tensor) else None)
    device, shape, dtype = q.device, q.shape, q.dtype
    dt = _DTYPES16.get(dtype)
    if dt is None:
        raise TypeError(f"q: dtype {dtype} is not supported (bfloat16, float16)")
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.device != device:
            _check_cuda(name, t, device)
        if t.dtype is not dtype:
            raise TypeError("k and v must have q's dtype")
    if len(shape) != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[2] != shape[2]:
        raise ValueError(f"q must be [T, H, D] and k, v [Tk, Hk, D], got {tuple(shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    T, H, D = shape
    Tk, Hk = k.shape[0], k.shape[1]
    if H == 0 or Hk == 0 or H % Hk:
        raise ValueError(f"{H} query heads are not a multiple of {Hk}")
    sums = []
    for name, t in (("cu_seqlens", cu_seqlens), ("cu_seqlens_k", cu_seqlens_k)):
        if t is None and name == "cu_seqlens_k":
            if Tk != T:
                raise ValueError(f"{Tk} keys for {T} queries need cu_seqlens_k")
            sums.append(None)
            continue
        n = t.shape[0] if isinstance(t, torch.Tensor) and t.dim() == 1 else 0
        if n == 0 or (sums and n != sums[0].shape[0]):
            raise ValueError(f"{name} must be a tensor of whole numbers [B + 1]")
        sums.append(_check_ids(name, t, n, device))
    if out is None:
        out = torch.empty(T, H, D, dtype=dtype, device=device)
    else:
        _check_cuda("out", out, device)
        if out.shape != shape or out.dtype != dtype:
            raise ValueError("out must match q's shape and dtype")
    index = device.index
    if index != _current_device():  # launches go to the current device
        with torch.cuda.device(index):
            return packed_attention(q, k, v, sums[0], sums[1], causal, scale, out=out)
    rc = _lib.load().wdrz_attn_packed(
        dt, q.data_ptr(), _lib.strides3(q.stride()), k.data_ptr(), _lib.strides3(k.stride()), v.data_ptr(),
        _lib.strides3(v.stride()), out.data_ptr(), _lib.strides3(out.stride()), sums[0].data_ptr(),
        None if sums[1] is None else sums[1].data_ptr(), sums[0].shape[0] - 1, T, Tk, H, Hk, D,
        D ** -0.5 if scale is None else scale, 1 if causal else 0, _raw_stream(index),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "packed_attention")
    return out


def scaled_dot_product_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    attn_mask: Optional[torch.Tensor] = None,
    dropout_p: float = 0.0,
    is_causal: bool = False,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """``F.scaled_dot_product_attention`` for ``[B, H, L, 64]`` inputs (reference ``model.py:288-296``).

    Inputs may be strided views (the reference passes rearranged ``[B, T, H*D]`` projections).
    The result is a ``[B, H, Lq, D]`` view of ``[B, Lq, H, D]`` storage, so the reference's
    ``rearrange(out, "B h T d -> B T (h d)")`` that follows is free. ``is_causal`` is torch's
    top-left aligned mask. ``attn_mask`` and dropout are not supported (the reference passes
    neither at inference).
    """
    if attn_mask is not None:
        raise NotImplementedError("attn_mask is not supported (the reference passes None)")
    if dropout_p != 0.0:
        raise NotImplementedError("dropout is not supported at inference")
    lib = _lib.load()
    device = query.device
    for name, t in (("query", query), ("key", key), ("value", value)):
        _check_cuda(name, t, device)
    if query.dim() != 4 or key.dim() != 4 or value.dim() != 4:
        raise ValueError("query/key/value must be 4-D [B, H, L, D]")
    B, H, Lq, D = query.shape
    Bk, Hk, Lk, Dk = key.shape
    if (Bk, Hk, Dk) != (B, H, D) or tuple(value.shape) != (B, H, Lk, D):
        raise ValueError(
            f"shape mismatch: query {tuple(query.shape)}, key {tuple(key.shape)}, value {tuple(value.shape)}"
        )
    dt = _dtype_code(query, "query")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError("query, key and value must share a dtype")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    out = torch.empty((B, Lq, H, D), dtype=query.dtype, device=device).permute(0, 2, 1, 3)
    if B == 0 or Lq == 0:
        return out
    if Lk == 0:
        raise ValueError("key length must be >= 1")
    rc = lib.wdrz_attn_fwd(
        dt,
        query.data_ptr(),
        key.data_ptr(),
        value.data_ptr(),
        out.data_ptr(),
        B, H, Lq, Lk, D,
        _lib.strides4(query.stride()),
        _lib.strides4(key.stride()),
        _lib.strides4(value.stride()),
        _lib.strides4(out.stride()),
        float(scale),
        int(bool(is_causal)),
        _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "scaled_dot_product_attention")
    return out


def qkv_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, n_head: int, causal: bool = False) -> torch.Tensor:
    """Attention core of ``MultiHeadAttention.qkv_attention`` (reference ``model.py:276-298``).

    ``q``, ``k``, ``v`` are the ``[B, T, n_head*64]`` projection outputs; returns
    ``[B, Tq, n_head*64]`` before the output projection. The scale is ``(D**-0.25)**2`` and the
    mask is causal only when ``causal and Tq > 1`` (``model.py:280-294``).
    """
    B, Tq, n_state = q.shape
    D = n_state // n_head
    scale = D ** -0.25
    qh = q.view(B, Tq, n_head, D).permute(0, 2, 1, 3)
    kh = k.view(k.shape[0], k.shape[1], n_head, D).permute(0, 2, 1, 3)
    vh = v.view(v.shape[0], v.shape[1], n_head, D).permute(0, 2, 1, 3)
    out = scaled_dot_product_attention(qh, kh, vh, is_causal=causal and Tq > 1, scale=scale * scale)
    return out.permute(0, 2, 1, 3).reshape(B, Tq, n_state)
