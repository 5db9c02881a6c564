"""Slot KV caches for the decoder, laid out for one MI355X (288 GB HBM3E).

``FlashKVCache`` keeps the reference's API (``src/whisperdrz/model.py:98-192``): buffers
``k_cache`` / ``v_cache`` indexed ``[slot, pos, head, dim]``, int32 ``seq_lens``, and the
methods ``prefill``, ``set_cross_attention`` and ``reset``. What changes is the storage:

* head-major: each cache is stored as ``[slot, head, pos, dim]`` and exposed as the permuted
  view ``[slot, pos, head, dim]`` that the reference indexes. A (slot, head) pair is then one
  contiguous run of ``pos * 128`` bytes, which is exactly what one attention workgroup streams;
  the attention kernels take strides, so they read the view directly.
* one arena for all layers: ``KVSlotPool`` carves every layer's self and cross caches out of a
  single allocation (2 MiB-aligned slices), so the decoder's 128 cache tensors are one
  allocation whose size is known up front, and ``plan_slots`` sizes the slot count for the
  HBM that is left after weights and activations.

* cache writes on the GPU go through ``wdrz_kv_fill`` (one kernel for K and V, contiguous 4 KB
  runs per (slot, head)) instead of torch's index_put over the permuted view, which is ~3x
  slower on the cross fill.

Sizes at Whisper large-v3 (32 layers, 20 heads, head_dim 64, bf16): 448-position self caches
take 73.4 MB per slot, 1500-position cross caches 245.8 MB per slot, 319 MB per slot in all;
about 850 slots fit in 272 GB. ``FlashKVCache8`` holds the same in 8 bits: 171 MB per slot, about 1590 slots.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch import Tensor

from . import _lib

_ALIGN = 2 << 20  # slice alignment inside the arena (bytes)
_FILL_DTYPES = {torch.bfloat16: _lib.WDRZ_BF16, torch.float16: _lib.WDRZ_F16}


def _hip_fill(k_cache: Tensor, v_cache: Tensor, k: Tensor, v: Tensor, slot_indices: Optional[Tensor],
              start_pos: int) -> bool:
    """``k_cache[slot_indices, start_pos:start_pos + T] = k`` (and v) with ``wdrz_kv_fill``.
    Returns False (nothing written) for what the kernel does not take: CPU tensors, a dtype
    other than the caches' bf16 / fp16, head_dim != 64; the caller then uses torch indexing,
    which also casts."""
    if not (k.is_cuda and k_cache.is_cuda and k.dtype == v.dtype == k_cache.dtype == v_cache.dtype
            and k.dtype in _FILL_DTYPES and k.shape[-1] == 64 and k.dim() == 4):
        return False
    from .attention import _raise, _stream_handle

    B, T, H, D = (int(x) for x in k.shape)
    if tuple(v.shape) != (B, T, H, D) or k_cache.shape[2] != H:
        raise ValueError(f"k/v {tuple(k.shape)} / {tuple(v.shape)} do not match the cache {tuple(k_cache.shape)}")
    if k.stride(-1) != 1 or v.stride() != k.stride():  # one set of source strides for both
        k, v = k.contiguous(), v.contiguous()
    slots = None
    if slot_indices is not None:
        slots = slot_indices.to(device=k.device, dtype=torch.int64)
        if slots.dim() != 1 or slots.shape[0] != B:
            raise ValueError(f"slot_indices must be [{B}]")
        slots = slots.contiguous()
    n_slots, Lmax = int(k_cache.shape[0]), int(k_cache.shape[1])
    rc = _lib.load().wdrz_kv_fill(
        _FILL_DTYPES[k.dtype], k.data_ptr(), v.data_ptr(), (_lib.ctypes.c_int64 * 3)(*k.stride()[:3]),
        k_cache.data_ptr(), v_cache.data_ptr(), (_lib.ctypes.c_int64 * 3)(*k_cache.stride()[:3]),
        slots.data_ptr() if slots is not None else None, B, T, H, D, n_slots, Lmax, int(start_pos),
        _stream_handle(),
    )
    if rc != _lib.WDRZ_OK:
        _raise(rc, "kv_fill")
    return True


class FlashKVCache:
    """Per-layer slot cache with the reference API (model.py:98-192), head-major storage.

    ``k_cache``/``v_cache`` are ``[batch_size, max_seq_length, n_heads, head_dim]`` views of
    ``[batch_size, n_heads, max_seq_length, head_dim]`` storage. Pass ``k_storage`` /
    ``v_storage`` (head-major tensors) to place the cache inside an existing arena.
    """

    def __init__(
        self,
        batch_size: int,
        max_seq_length: int,
        n_heads: int,
        head_dim: int,
        dtype=torch.float16,
        device=None,
        *,
        k_storage: Optional[Tensor] = None,
        v_storage: Optional[Tensor] = None,
        seq_lens: Optional[Tensor] = None,
    ):
        self.batch_size = batch_size
        self.max_seq_length = max_seq_length
        self.n_heads = n_heads
        self.head_dim = head_dim
        shape_hm = (batch_size, n_heads, max_seq_length, head_dim)
        if k_storage is None:
            k_storage = torch.zeros(shape_hm, dtype=dtype, device=device)
            v_storage = torch.zeros(shape_hm, dtype=dtype, device=device)
        if tuple(k_storage.shape) != shape_hm or tuple(v_storage.shape) != shape_hm:
            raise ValueError(f"storage must have head-major shape {shape_hm}")
        self.k_storage = k_storage
        self.v_storage = v_storage
        self.k_cache = k_storage.permute(0, 2, 1, 3)
        self.v_cache = v_storage.permute(0, 2, 1, 3)
        if seq_lens is None:
            seq_lens = torch.zeros(batch_size, dtype=torch.int32, device=k_storage.device)
        self.seq_lens = seq_lens
        self.done = False
        self.cross_attn_len = 0

    @property
    def dtype(self) -> torch.dtype:
        return self.k_storage.dtype

    @property
    def device(self) -> torch.device:
        return self.k_storage.device

    def prefill(self, k: Tensor, v: Tensor, start_pos: int = 0, slot_indices: Optional[Tensor] = None):
        """Write ``k, v`` ``[B, seq, heads, head_dim]`` at ``start_pos`` and set ``seq_lens``
        to the end position (model.py:150-168)."""
        seq_len = k.shape[1]
        end_pos = start_pos + seq_len
        written = _hip_fill(self.k_cache, self.v_cache, k, v, slot_indices, start_pos)
        if slot_indices is not None:
            if not written:
                self.k_cache[slot_indices, start_pos:end_pos] = k
                self.v_cache[slot_indices, start_pos:end_pos] = v
            self.seq_lens[slot_indices] = end_pos
        else:
            B = k.shape[0]
            if not written:
                self.k_cache[:B, start_pos:end_pos] = k
                self.v_cache[:B, start_pos:end_pos] = v
            self.seq_lens[:B] = end_pos

    def set_cross_attention(self, k: Tensor, v: Tensor, slot_indices: Optional[Tensor] = None):
        """Write the encoder-side ``k, v`` ``[B, seq, heads, head_dim]`` (model.py:170-183)."""
        seq_len = k.shape[1]
        if not _hip_fill(self.k_cache, self.v_cache, k, v, slot_indices, 0):
            if slot_indices is not None:
                self.k_cache[slot_indices, :seq_len] = k
                self.v_cache[slot_indices, :seq_len] = v
            else:
                B = k.shape[0]
                self.k_cache[:B, :seq_len] = k
                self.v_cache[:B, :seq_len] = v
        self.cross_attn_len = seq_len
        self.done = True

    def reset(self, slot_indices: Optional[Tensor] = None):
        """Zero the lengths of ``slot_indices`` (all slots if None); K/V are not cleared
        (model.py:185-192)."""
        if slot_indices is not None:
            self.seq_lens[slot_indices] = 0
        else:
            self.seq_lens.zero_()
        self.done = False
        self.cross_attn_len = 0


class FlashKVCache8:
    """The slot cache held in 8 bits: ``FlashKVCache``'s methods over e4m3 codes, for
    ``flash_attn_with_kvcache8``.

    Positions are held in blocks of 32; a complete block of one (slot, head) is codes with one power-of-two
    scale for its keys and one for its values (:meth:`dequantize` says what they stand for). With ``ring``
    (a self cache) the newest positions also stand as they came, in 64 rows a (slot, head), and the block
    that is not complete is read from there: a position is rounded once, when its block completes, however
    the tokens were cut into calls. A slot's length may be set back to 32 below the furthest position that
    was written (a draft that was rejected), or to any multiple of 32, from where that count starts anew;
    anywhere else the ring's rows are others.
    Without ``ring`` (a cross cache) the cache is filled by :meth:`set_cross_attention`.

    Buffers: ``k_codes`` / ``v_codes`` ``[batch_size, n_heads, blocks * 32, 64]`` (``float8_e4m3fn``),
    ``k_scales`` / ``v_scales`` ``[batch_size, n_heads, blocks]`` fp32, ``k_ring`` / ``v_ring``
    ``[batch_size, n_heads, 64, 64]`` of ``dtype``; ``storage`` places them in given (contiguous) tensors, which
    the cache then keeps. Scales are powers of two. Blocks that nobody has written stand for zeros in buffers of zeros.
    Per slot and head 128 bytes a position and 16 KB of ring, against 256 bytes a position in 16 bits.
    """

    BLOCK = 32
    RING = 64

    def __init__(self, batch_size: int, max_seq_length: int, n_heads: int, head_dim: int = 64, dtype=torch.bfloat16,
                 device=None, *, ring: bool = True, storage: Optional[dict[str, Tensor]] = None,
                 seq_lens: Optional[Tensor] = None):
        layout = self.layout(batch_size, max_seq_length, n_heads, dtype, ring, head_dim)
        self.batch_size, self.max_seq_length = batch_size, max_seq_length
        self.n_heads, self.head_dim, self.dtype, self.has_ring = n_heads, head_dim, dtype, bool(ring)
        if storage is None:
            storage = {n: torch.zeros(shape, dtype=torch.uint8, device=device).view(dt) if dt is torch.float8_e4m3fn
                       else torch.zeros(shape, dtype=dt, device=device) for n, (shape, dt) in layout.items()}
        for n, (shape, dt) in layout.items():
            t = storage.get(n)
            if t is None or tuple(t.shape) != shape or t.dtype != dt or not t.is_contiguous():
                raise ValueError(f"storage[{n!r}] must be a contiguous {dt} tensor of shape {shape}")
            if t.device != storage["k_codes"].device:
                raise ValueError("the buffers must be on one device")
            setattr(self, n, t)
        if not ring:
            self.k_ring = self.v_ring = None
        self.device = self.k_codes.device
        self._held = tuple(storage[n] for n in layout)  # the kernels' pointers are these tensors', whatever the attributes become
        self.struct = _lib.Kv8(*(storage[n].data_ptr() if n in layout else None for n in
                                 ("k_codes", "v_codes", "k_scales", "v_scales", "k_ring", "v_ring")),
                               batch_size, n_heads, max_seq_length)
        self.seq_lens = torch.zeros(batch_size, dtype=torch.int32, device=self.device) if seq_lens is None else seq_lens
        self.done = False
        self.cross_attn_len = 0

    @classmethod
    def layout(cls, batch_size: int, max_seq_length: int, n_heads: int, dtype, ring: bool, head_dim: int = 64) -> dict:
        """Shape and dtype of every buffer."""
        if head_dim != 64:
            raise NotImplementedError(f"head_dim {head_dim} is not supported (only 64)")
        if dtype not in _FILL_DTYPES:
            raise TypeError(f"dtype {dtype} is not supported (bfloat16, float16)")
        blocks = -(-max_seq_length // cls.BLOCK)
        res = {}
        for n in "kv":
            res[n + "_codes"] = ((batch_size, n_heads, blocks * cls.BLOCK, 64), torch.float8_e4m3fn)
            res[n + "_scales"] = ((batch_size, n_heads, blocks), torch.float32)
            if ring:
                res[n + "_ring"] = ((batch_size, n_heads, cls.RING, 64), dtype)
        return res

    def _write(self, k: Tensor, v: Tensor, slot_indices: Optional[Tensor], start_pos: int) -> None:
        from .attention import _check_cuda, _current_device, _raise, _raw_stream

        _check_cuda("k", k, self.device)
        _check_cuda("v", v, self.device)
        if k.dim() != 4 or k.shape[2:] != (self.n_heads, self.head_dim) or v.shape != k.shape:
            raise ValueError(f"k and v must be [B, T, {self.n_heads}, {self.head_dim}], got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.dtype not in _FILL_DTYPES or v.dtype != k.dtype or (self.has_ring and k.dtype != self.dtype):
            raise TypeError(f"k and v: dtypes {k.dtype} and {v.dtype} do not match the cache's")
        B, T = k.shape[0], k.shape[1]
        slots = None
        if slot_indices is not None:
            _check_cuda("slot_indices", slot_indices, self.device)
            if slot_indices.is_floating_point() or slot_indices.shape != (B,):
                raise ValueError(f"slot_indices must be whole numbers [{B}]")
            slots = slot_indices.to(torch.int64).contiguous()
        if B == 0 or T == 0:
            return
        index = self.device.index
        if index != _current_device():  # launches go to the current device
            with torch.cuda.device(index):
                return self._write(k, v, slots, start_pos)
        rc = _lib.load().wdrz_kv8_write(
            _FILL_DTYPES[k.dtype], self.struct, k.data_ptr(), _lib.strides(k.stride()), v.data_ptr(),
            _lib.strides(v.stride()), None if slots is None else slots.data_ptr(), B, T, start_pos, _raw_stream(index))
        if rc != _lib.WDRZ_OK:
            _raise(rc, "kv8_write")

    def prefill(self, k: Tensor, v: Tensor, start_pos: int = 0, slot_indices: Optional[Tensor] = None):
        """Append ``k, v`` ``[B, seq, heads, 64]`` at length ``start_pos`` and set ``seq_lens`` to the end."""
        if not self.has_ring:
            raise ValueError("prefill needs a cache with a ring")
        self._write(k, v, slot_indices, start_pos)
        if slot_indices is not None:
            self.seq_lens[slot_indices] = start_pos + k.shape[1]
        else:
            self.seq_lens[: k.shape[0]] = start_pos + k.shape[1]

    def set_cross_attention(self, k: Tensor, v: Tensor, slot_indices: Optional[Tensor] = None):
        """Fill the slots with the encoder-side ``k, v`` ``[B, seq, heads, 64]``."""
        if self.has_ring:
            raise ValueError("set_cross_attention needs a cache without a ring")
        self._write(k, v, slot_indices, 0)
        self.cross_attn_len = k.shape[1]
        self.done = True

    def dequantize(self, lengths: Optional[Tensor] = None) -> tuple[Tensor, Tensor]:
        """fp32 ``[batch_size, max_seq_length, n_heads, 64]`` keys and values of every slot, as the attention
        reads them at ``lengths`` ``[batch_size]`` (``seq_lens`` if None; a cache without a ring has none)."""
        L, res = self.max_seq_length, []
        pos = torch.arange(L, device=self.device)
        for codes, scales, ring in ((self.k_codes, self.k_scales, self.k_ring), (self.v_codes, self.v_scales, self.v_ring)):
            x = codes.float()[:, :, :L] * scales.repeat_interleave(self.BLOCK, -1)[:, :, :L, None]
            if ring is not None:
                n = self.seq_lens if lengths is None else lengths
                x = torch.where((pos < (n // self.BLOCK * self.BLOCK)[:, None])[:, None, :, None], x,
                                ring.float()[:, :, pos % self.RING])
            res.append(x.permute(0, 2, 1, 3))
        return res[0], res[1]

    def reset(self, slot_indices: Optional[Tensor] = None):
        """Zero the lengths of ``slot_indices`` (all slots if None); nothing is cleared."""
        if slot_indices is not None:
            self.seq_lens[slot_indices] = 0
        else:
            self.seq_lens.zero_()
        self.done = False
        self.cross_attn_len = 0


@dataclass(frozen=True)
class SlotPlan:
    n_slots: int
    bytes_per_slot: int
    total_bytes: int


def _cache_buffers(n_slots: int, n_heads: int, head_dim: int, seq_len: int, dtype: torch.dtype, bits: int,
                   ring: bool) -> dict[str, tuple[tuple[int, ...], torch.dtype]]:
    """Shape and dtype of every buffer of one cache, 16-bit (``dtype``'s, head-major) or 8-bit."""
    if bits == 8:
        return FlashKVCache8.layout(n_slots, seq_len, n_heads, dtype, ring, head_dim)
    if bits != 16:
        raise ValueError(f"cache_bits {bits} is not 16 (dtype's) or 8")
    return {n: ((n_slots, n_heads, seq_len, head_dim), dtype) for n in ("k_storage", "v_storage")}


def _buffer_bytes(shape: tuple[int, ...], dtype: torch.dtype) -> int:
    n = torch.empty((), dtype=dtype).element_size()
    for x in shape:
        n *= x
    return n


def cache_bytes_per_slot(n_layers: int, n_heads: int, head_dim: int, self_len: int, cross_len: int,
                         dtype: torch.dtype, cache_bits: int = 16) -> int:
    return n_layers * sum(_buffer_bytes(*b) for length, ring in ((self_len, True), (cross_len, False))
                          for b in _cache_buffers(1, n_heads, head_dim, length, dtype, cache_bits, ring).values())


def plan_slots(hbm_budget_bytes: int, n_layers: int = 32, n_heads: int = 20, head_dim: int = 64,
               self_len: int = 448, cross_len: int = 1500, dtype: torch.dtype = torch.bfloat16,
               cache_bits: int = 16) -> SlotPlan:
    """How many decode slots a KV arena of ``hbm_budget_bytes`` holds at these sizes."""
    per = cache_bytes_per_slot(n_layers, n_heads, head_dim, self_len, cross_len, dtype, cache_bits)
    # every per-layer slice is rounded up to the arena alignment
    n = max(0, hbm_budget_bytes // per)
    size = lambda n: KVSlotPool.arena_bytes(n, n_layers, n_heads, head_dim, self_len, cross_len, dtype, cache_bits)
    while n > 0 and size(n) > hbm_budget_bytes:
        n -= 1
    return SlotPlan(n_slots=int(n), bytes_per_slot=per, total_bytes=size(n))


class KVSlotPool:
    """All layers' self and cross caches in one arena (replaces ``create_flash_kv``,
    model.py:773-808, and ``reset_flash_kv``, model.py:810-822).

    ``self_kv[l]`` / ``cross_kv[l]`` are ``FlashKVCache`` objects whose storage are slices of
    the arena. Self caches of all layers share nothing but the arena; each layer keeps its
    own ``seq_lens`` as in the reference, stored as row ``l`` of one ``[n_layers, n_slots]``
    int32 tensor (``self_seq_lens``) so that a decode step can gather and bump every layer's
    lengths with one operation each.

    ``cache_bits=8`` holds the caches in 8 bits (``FlashKVCache8``, the self caches with a ring): 171 MB a slot
    at large-v3 instead of 319 MB. ``dtype`` is then the activations'.
    """

    def __init__(self, n_layers: int, n_slots: int, n_heads: int = 20, head_dim: int = 64,
                 self_len: int = 448, cross_len: int = 1500, dtype: torch.dtype = torch.bfloat16,
                 device=None, cache_bits: int = 16):
        self.n_layers, self.n_slots = n_layers, n_slots
        self.n_heads, self.head_dim = n_heads, head_dim
        self.self_len, self.cross_len = self_len, cross_len
        self.dtype = dtype
        self.cache_bits = cache_bits
        nbytes = self.arena_bytes(n_slots, n_layers, n_heads, head_dim, self_len, cross_len, dtype, cache_bits)
        self.arena = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        off = 0

        def cache(seq_len: int, ring: bool, seq_lens: Optional[Tensor]):
            nonlocal off
            st = {}
            for name, (shape, dt) in _cache_buffers(n_slots, n_heads, head_dim, seq_len, dtype, cache_bits, ring).items():
                n = _buffer_bytes(shape, dt)
                st[name] = self.arena[off : off + n].view(dt).view(shape)
                off += (n + _ALIGN - 1) // _ALIGN * _ALIGN
            if cache_bits == 8:
                return FlashKVCache8(n_slots, seq_len, n_heads, head_dim, dtype, ring=ring, storage=st, seq_lens=seq_lens)
            return FlashKVCache(n_slots, seq_len, n_heads, head_dim, seq_lens=seq_lens, **st)

        self.self_kv: list = []
        self.cross_kv: list = []
        self.self_seq_lens = torch.zeros((n_layers, n_slots), dtype=torch.int32, device=self.arena.device)
        for l in range(n_layers):
            self.self_kv.append(cache(self_len, True, self.self_seq_lens[l]))
            self.cross_kv.append(cache(cross_len, False, None))

    @property
    def device(self) -> torch.device:
        return self.arena.device

    @staticmethod
    def arena_bytes(n_slots: int, n_layers: int, n_heads: int, head_dim: int, self_len: int, cross_len: int,
                    dtype: torch.dtype, cache_bits: int = 16) -> int:
        rounded = lambda b: (_buffer_bytes(*b) + _ALIGN - 1) // _ALIGN * _ALIGN
        return n_layers * sum(rounded(b) for length, ring in ((self_len, True), (cross_len, False))
                              for b in _cache_buffers(n_slots, n_heads, head_dim, length, dtype, cache_bits, ring).values())

    def reset(self, slot_indices: Optional[Tensor] = None) -> None:
        for s_kv, c_kv in zip(self.self_kv, self.cross_kv, strict=True):
            s_kv.reset(slot_indices)
            c_kv.reset(slot_indices)
